"""Per-head RMSNorm of queries and keys with the position rotation, in one
pass over fused QKV rows.

The reference leaves both to its mlx_lm models; here they are one kernel
(``cq_qk_norm_rope_rows``) between a model's QKV projection and the cache:
``decoder.Qwen3StyleDecoder.prefill`` runs its prompts through it.
"""

from __future__ import annotations

import torch

from . import _lib
from .trace import traced
from ._tensors import cq_dtype, on_device, require_cuda, stream_ptr


@traced("cq.qk_norm_rope")
def qk_norm_rope(qkv: torch.Tensor, n_q_heads: int, n_kv_heads: int, inv_freq: torch.Tensor, positions: torch.Tensor,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, *, eps: float = 1e-6,
                 pairs: str = "halves"):
    """Queries [B, Hq, S, D] and keys [B, Hkv, S, D] of fused rows ``qkv`` [B,
    S, (Hq + 2 Hkv) * D] (heads q | k | v; values are not touched: they are the
    last Hkv * D columns).

    Each q and k head is RMS-normalised over its channels and weighted
    (``q_weight`` / ``k_weight`` [D]; both None: no norm), then its first 2 *
    len(inv_freq) channels are rotated by ``positions * inv_freq`` -- positions
    int64, broadcastable to [B, S]; inv_freq fp32 -- as pairs (i, i + half)
    (``pairs="halves"``) or (2i, 2i + 1) (``"adjacent"``).  fp32 arithmetic,
    one rounding to qkv's dtype (float16, bfloat16 or float32)."""
    shape, dev = qkv.shape, qkv.device
    if len(shape) != 3:
        raise ValueError(f"qk_norm_rope: qkv must be [B, S, (Hq + 2 Hkv) * D], got {tuple(shape)}")
    B, S, width = shape
    heads = n_q_heads + 2 * n_kv_heads
    if n_q_heads < 1 or n_kv_heads < 1 or width == 0 or width % heads:
        raise ValueError(f"qk_norm_rope: rows of {width} do not hold {n_q_heads} + 2 * {n_kv_heads} heads")
    D = width // heads
    if pairs not in ("halves", "adjacent"):
        raise ValueError(f"qk_norm_rope: pairs must be 'halves' or 'adjacent', got {pairs!r}")
    require_cuda(qkv)
    dt = cq_dtype(qkv)
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or inv_freq.device != dev:
        raise ValueError(f"qk_norm_rope: inv_freq must be fp32 [rot / 2] on {dev}")
    half = inv_freq.shape[0]
    if 2 * half > D:
        raise ValueError(f"qk_norm_rope: {half} frequencies rotate more than {D} channels")
    if positions.dtype != torch.int64 or positions.device != dev:
        raise ValueError(f"qk_norm_rope: positions must be int64 on {dev}")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("qk_norm_rope: give both norm weights or neither")
    wq = wk = None
    if q_weight is not None:
        for w in (q_weight, k_weight):
            if w.shape != (D,) or w.dtype != qkv.dtype or w.device != dev:
                raise ValueError(f"qk_norm_rope: norm weights must be {qkv.dtype} [{D}] on {dev}")
        q_weight, k_weight = q_weight.contiguous(), k_weight.contiguous()
        wq, wk = q_weight.data_ptr(), k_weight.data_ptr()
    if positions.shape != (B, S):
        positions = positions.expand(B, S)
    strides = qkv.stride()
    if strides[2] != 1:
        qkv = qkv.contiguous()
        strides = qkv.stride()
    inv_freq = inv_freq.contiguous()
    pb, ps = positions.stride()
    q = qkv.new_empty((B, n_q_heads, S, D))
    k = qkv.new_empty((B, n_kv_heads, S, D))
    with on_device(dev):
        _lib.check(_lib.lib().cq_qk_norm_rope_rows(
            qkv.data_ptr(), strides[0], strides[1], B, S, n_q_heads, n_kv_heads, D, 2 * half,
            1 if pairs == "adjacent" else 0, wq, wk, inv_freq.data_ptr(), positions.data_ptr(), pb, ps, float(eps),
            q.data_ptr(), k.data_ptr(), dt, stream_ptr(dev)), "qk_norm_rope")
    return q, k
