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
    one rounding to qkv's dtype (float16, bfloat16 or float32); angles keep
    their phase for positions up to 2^53.  No gradients, as everywhere in this
    package: the results are detached whatever qkv and the weights require."""
    if pairs not in ("halves", "adjacent"):
        raise ValueError(f"qk_norm_rope: pairs must be 'halves' or 'adjacent', got {pairs!r}")
    return _lib.calls().qk_norm_rope(qkv, n_q_heads, n_kv_heads, inv_freq, positions, q_weight, k_weight, eps,
                                     pairs == "adjacent")
