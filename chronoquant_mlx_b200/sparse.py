"""Sparse attention over a compressed cache: every query token attends to the
blocks of tokens that a cheap score picks for it, so a decode step reads
``top`` blocks of the history instead of all of it.

The reference attends to the whole history (attention.py:23-74); this is an
addition around the same cache.  Three steps, each on the caller's stream::

    index = BlockIndex(cache, block_tokens=64)      # beside the cache
    cache.update_and_fetch(keys, values)
    index.update()                                  # summarise what is new
    blocks = index.select(queries, top=64, first=1, recent=2)
    out = chronoquant_sparse_sdpa(queries, cache, scale, blocks, index.block_tokens)

``BlockIndex`` keeps, per block and kv-head, the range of the decoded keys'
channels in 8 bits (2 * head_dim + 4 bytes a block); ``select`` scores every
block by the largest q.k its ranges allow and lists the best ones per query
token; the attention kernel reads the listed blocks of the paged cache
directly.  Queries are the newest tokens of the cache: query i of q_len sits at
position offset - q_len + i and sees nothing behind it.  ``starts`` gives the
first real token of each sequence of a left-padded batch; a row that sees no
token gets zeros.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .trace import traced
from ._tensors import on_device, require_cuda, stream_ptr

MAX_TOP = 4096  # longest block list


_QUERY_DT = {torch.float16: _lib.CQ_F16, torch.bfloat16: _lib.CQ_BF16}


def _check_queries(q: torch.Tensor, st, T: int, what: str):
    """(queries with contiguous channels, C dtype, Hq, Tq, strides) after the checks against a store."""
    shape = q.shape
    if len(shape) != 4 or shape[0] != st.B or shape[3] != st.D:
        raise ValueError(f"{what}: queries must be [{st.B}, Hq, Tq, {st.D}], got {tuple(shape)}")
    if q.device != st.device:
        require_cuda(q)
        raise ValueError(f"{what}: queries on {q.device}, the cache on {st.device}")
    dt = _QUERY_DT.get(q.dtype)
    if dt is None:
        raise TypeError(f"{what}: queries must be float16 or bfloat16, got {q.dtype}")
    _, Hq, S, _ = shape
    if Hq == 0 or Hq % st.H:
        raise ValueError(f"{what}: {Hq} query heads are no multiple of {st.H} kv-heads")
    if not 1 <= S <= T:
        raise ValueError(f"{what}: {S} query tokens, {T} tokens cached")
    strides = q.stride()
    if strides[3] != 1:
        q = q.contiguous()
        strides = q.stride()
    return q, dt, Hq, S, strides


def _check_starts(starts, B: int, device, what: str):
    if starts is None:
        return None
    if starts.dtype != torch.int64 or starts.shape != (B,) or starts.device != device:
        raise ValueError(f"{what}: starts must be int64 [{B}] on {device}, got {starts.dtype} {tuple(starts.shape)} "
                         f"on {starts.device}")
    return starts if starts.is_contiguous() else starts.contiguous()


class BlockIndex:
    """Per-block key ranges of one ``ChronoQuantCache`` and the selection of
    blocks by them.

    ``block_tokens``: tokens per block, a multiple of 16 (64 suits the cache's
    chunk sizes).  ``codes`` int8 [B, Hkv, capacity, 2, D] and ``scales`` fp32
    [B, Hkv, capacity] follow the cache's page pool; ``covered`` is the number
    of tokens summarised."""

    def __init__(self, cache, block_tokens: int = 64):
        if int(block_tokens) < 16 or int(block_tokens) % 16:
            raise ValueError(f"block_tokens must be a positive multiple of 16, got {block_tokens}")
        self.cache = cache
        self.block_tokens = int(block_tokens)
        self.codes = None
        self.scales = None
        self.covered = 0
        self._store = None

    @property
    def n_blocks(self) -> int:
        """Blocks summarised so far (the last one may be partial)."""
        return -(-self.covered // self.block_tokens)

    @property
    def nbytes(self) -> int:
        return 0 if self.codes is None else self.codes.numel() + self.scales.numel() * 4

    def reserve(self, tokens: int) -> None:
        """Room for ``tokens`` tokens per sequence (and for all the cache's pool maps)."""
        st = self.cache.store
        if st is None:
            raise ValueError("BlockIndex: the cache is empty")
        if st is not self._store:  # another store (a restored state): nothing of the old ranges holds
            self._store, self.codes, self.scales, self.covered = st, None, None, 0
        need = -(-max(int(tokens), st.capacity_tokens()) // self.block_tokens)
        have = 0 if self.codes is None else self.codes.shape[2]
        if need <= have:
            return
        codes = torch.zeros((st.B, st.H, need, 2, st.D), dtype=torch.int8, device=st.device)
        scales = torch.zeros((st.B, st.H, need), dtype=torch.float32, device=st.device)
        if have:
            codes[:, :, :have].copy_(self.codes)
            scales[:, :, :have].copy_(self.scales)
        self.codes, self.scales = codes, scales

    @traced("cq.block_bounds")
    def update(self, start: int | None = None) -> "BlockIndex":
        """Summarise the blocks that hold tokens from ``start`` on (default:
        what was appended since the last update).  Returns the index."""
        c = self.cache
        T = c.offset
        st = c.store
        if T == 0 or st is None:
            raise ValueError("BlockIndex: the cache is empty")
        if st is not self._store or self.codes.shape[2] * self.block_tokens < st.capacity_tokens():
            self.reserve(T)
        t0 = self.covered if start is None else int(start)
        if not 0 <= t0 <= T:
            raise ValueError(f"BlockIndex: start {t0} outside [0, {T}]")
        t0 = min(t0, self.covered)
        with on_device(st.device):
            _lib.check(_lib.lib().cq_block_bounds(ctypes.byref(st.descriptor()), t0, T, self.block_tokens,
                                                  self.codes.data_ptr(), self.scales.data_ptr(), self.codes.shape[2],
                                                  stream_ptr(st.device)), "BlockIndex.update")
        self.covered = T
        return self

    def bounds(self, first: int = 0) -> torch.Tensor:
        """The key ranges of blocks ``first`` on: fp32 [B, Hkv, n, 2, D],
        lower bounds at index 0 and upper bounds at index 1 of dim 3."""
        n = self.n_blocks - int(first)
        if first < 0 or n < 0 or self.codes is None:
            raise ValueError(f"BlockIndex: first block {first} outside [0, {self.n_blocks}] (or nothing summarised)")
        st = self._store
        out = torch.empty((st.B, st.H, n, 2, st.D), dtype=torch.float32, device=st.device)
        with on_device(st.device):
            _lib.check(_lib.lib().cq_block_bounds_read(self.codes.data_ptr(), self.scales.data_ptr(), st.B * st.H,
                                                       self.codes.shape[2], first, n, st.D, out.data_ptr(),
                                                       stream_ptr(st.device)), "BlockIndex.bounds")
        return out

    @traced("cq.block_select")
    def select(self, queries: torch.Tensor, top: int, *, first: int = 1, recent: int = 2, starts=None,
               return_scores: bool = False):
        """Up to ``top`` blocks for every query token of ``queries`` [B, Hq,
        Tq, D] (the cache's newest tokens) and kv-head: int32 [B, Hkv, Tq,
        top], ascending, -1 behind.  The ``first`` lowest and ``recent`` highest
        blocks a token may see are always listed, the others by score (ties to
        the lower index).  ``starts``: int64 [B], first real token of each
        sequence.  ``return_scores``: also the listed blocks' scores (fp32, -inf
        behind), by which lists of ranks that share a sequence can be merged."""
        if not 1 <= top <= MAX_TOP or first < 0 or recent < 0 or first + recent > top:
            raise ValueError(f"select: need 1 <= top <= {MAX_TOP} and first + recent <= top, got top={top}, "
                             f"first={first}, recent={recent}")
        if self.covered != self.cache.offset or self.cache.store is not self._store or self.covered == 0:
            self.update()
        st, T = self._store, self.covered
        q, dt, Hq, S, (sb, sh, sq, _) = _check_queries(queries, st, T, "select")
        starts = _check_starts(starts, st.B, st.device, "select")
        B, H, bt = st.B, st.H, self.block_tokens
        row = -(-T // bt) + 7 & ~7  # a score row: cq_block_select_workspace, without the call
        ws = q.new_empty((B * H * S * row,), dtype=torch.float32)
        blocks = q.new_empty((B, H, S, top), dtype=torch.int32)
        scores = torch.empty_like(blocks, dtype=torch.float32) if return_scores else None
        with on_device(st.device):
            _lib.check(_lib.lib().cq_block_select(
                self.codes.data_ptr(), self.scales.data_ptr(), self.codes.shape[2], bt, B, H, st.D, T, None,
                q.data_ptr(), dt, Hq, S, sb, sh, sq, None if starts is None else starts.data_ptr(), first, recent, top,
                blocks.data_ptr(), None if scores is None else scores.data_ptr(), ws.data_ptr(), ws.numel() * 4,
                stream_ptr(st.device)), "select")
        return (blocks, scores) if return_scores else blocks


def _attention_workspace(st, d, T: int, Hq: int, S: int, top: int, bt: int) -> int:
    """cq_sparse_attention_workspace, kept per store: it depends on these numbers and the store's layout alone."""
    sizes = st.__dict__.setdefault("_sparse_ws", {})
    need = sizes.get((Hq, S, top, bt))
    if need is None:
        n = ctypes.c_size_t(0)
        _lib.check(_lib.lib().cq_sparse_attention_workspace(d, T, Hq, S, top, bt, ctypes.byref(n)),
                   "chronoquant_sparse_sdpa")
        need = sizes[Hq, S, top, bt] = n.value
    return need


@traced("cq.sparse_sdpa")
def chronoquant_sparse_sdpa(queries: torch.Tensor, cache, scale: float, blocks: torch.Tensor, block_tokens: int, *,
                            starts=None, return_lse: bool = False):
    """Attention of ``queries`` [B, Hq, Tq, D] (fp16/bf16, the cache's newest
    tokens) over the tokens of the listed blocks: ``blocks`` int32 [B, Hkv, Tq,
    n], ascending as ``BlockIndex.select`` lists them (an entry that is negative
    or not above its predecessor is left out).  Returns [B, Hq, Tq, D] in the
    query dtype; with ``return_lse`` an fp32 output and the fp32 log-sum-exp [B,
    Hq, Tq] (-inf for a row that sees no token), for merging."""
    st, T = cache.store, cache.offset
    if st is None or T == 0:
        raise ValueError("chronoquant_sparse_sdpa: the cache is empty")
    q, dt, Hq, S, (sb, sh, sq, _) = _check_queries(queries, st, T, "chronoquant_sparse_sdpa")
    B, H, dev = st.B, st.H, st.device
    shape = blocks.shape
    if len(shape) != 4 or shape[0] != B or shape[1] != H or shape[2] != S or blocks.dtype != torch.int32:
        raise ValueError(f"chronoquant_sparse_sdpa: blocks must be int32 [{B}, {H}, {S}, n], got {blocks.dtype} "
                         f"{tuple(shape)}")
    if blocks.device != dev:
        raise ValueError(f"chronoquant_sparse_sdpa: blocks on {blocks.device}, the cache on {dev}")
    top = shape[3]
    if not 1 <= top <= MAX_TOP:
        raise ValueError(f"chronoquant_sparse_sdpa: lists of 1 to {MAX_TOP} blocks, got {top}")
    if int(block_tokens) < 16 or int(block_tokens) % 16:
        raise ValueError(f"block_tokens must be a positive multiple of 16, got {block_tokens}")
    starts = _check_starts(starts, B, dev, "chronoquant_sparse_sdpa")
    if not blocks.is_contiguous():
        blocks = blocks.contiguous()
    d = ctypes.byref(st.descriptor())
    if return_lse:
        out = q.new_empty((B, Hq, S, st.D), dtype=torch.float32)
        lse = q.new_empty((B, Hq, S), dtype=torch.float32)
    else:
        out, lse = q.new_empty((B, Hq, S, st.D)), None
    with on_device(dev):
        need = _attention_workspace(st, d, T, Hq, S, top, block_tokens)
        ws = q.new_empty((need,), dtype=torch.uint8) if need else None
        _lib.check(_lib.lib().cq_sparse_attention(
            d, T, None, q.data_ptr(), dt, Hq, S, sb, sh, sq, float(scale), None if starts is None else
            starts.data_ptr(), blocks.data_ptr(), top, block_tokens, out.data_ptr(), _lib.CQ_F32 if return_lse else dt,
            None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(), need, stream_ptr(dev)),
            "chronoquant_sparse_sdpa")
    return (out, lse) if return_lse else out
