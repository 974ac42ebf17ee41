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
directly.  Lists hold at most 4096 blocks.  Queries are the newest tokens of the
cache: query i of q_len sits at position offset - q_len + i and sees nothing
behind it.  ``starts`` gives the first real token of each sequence of a
left-padded batch; a row that sees no token gets zeros.  The lengths are the
host's: a call captured into a CUDA graph replays at the length it was captured
at (``decoder.Qwen3StyleDecoder(sparse=...)`` captures steps that read the length
from device memory).
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .trace import traced


class BlockIndex:
    """Per-block key ranges of one ``ChronoQuantCache`` and the selection of
    blocks by them.

    ``block_tokens``: tokens per block, a multiple of 16 (64 suits the cache's
    chunk sizes).  ``codes`` int8 [B, Hkv, capacity, 2, D] and ``scales`` fp32
    [B, Hkv, capacity] follow the cache's page pool; ``covered`` is the number
    of tokens summarised.

    An update recorded into a CUDA graph counts for the calls of that capture;
    ``covered`` stays what it was, and what comes later summarises those tokens
    for itself.  A replay summarises the tokens of its capture: after the cache
    has grown it leaves the last of their blocks short, until ``update(start)``
    from that length.  ``reserve`` room before a capture: growing moves the
    tensors, which a graph's replays would not follow."""

    def __init__(self, cache, block_tokens: int = 64):
        if int(block_tokens) < 16 or int(block_tokens) % 16:
            raise ValueError(f"block_tokens must be a positive multiple of 16, got {block_tokens}")
        self.cache = cache
        self.block_tokens = int(block_tokens)
        self.codes = None
        self.scales = None
        self.covered = 0
        self._recorded = None  # (capture, tokens) of the last update that a capture recorded
        self._store = None

    def _tokens(self) -> int:
        """Tokens summarised for the next call: ``covered``, or what the capture it is recorded by recorded before."""
        if self._recorded is not None and self._recorded[0] == _lib.calls().capture_of(self.codes):
            return self._recorded[1]
        return self.covered

    @property
    def n_blocks(self) -> int:
        """Blocks summarised so far (the last one may be partial)."""
        return -(-self._tokens() // self.block_tokens)

    @property
    def nbytes(self) -> int:
        return 0 if self.codes is None else self.codes.numel() + self.scales.numel() * 4

    def reserve(self, tokens: int) -> None:
        """Room for ``tokens`` tokens per sequence (and for all the cache's pool maps)."""
        st = self.cache.store
        if st is None:
            raise ValueError("BlockIndex: the cache is empty")
        other = st is not self._store  # a restored state: nothing of the old ranges holds
        need = -(-max(int(tokens), st.capacity_tokens()) // self.block_tokens)
        have = 0 if other or self.codes is None else self.codes.shape[2]
        if need <= have:
            return
        with torch.cuda.device(st.device):
            recorded = torch.cuda.is_current_stream_capturing()
        if have and recorded:
            raise RuntimeError("BlockIndex: the index has to grow, which a capture cannot record; reserve() before it")
        # in a capture no zeros either: a replay would write them over ranges summarised since
        new = torch.empty if recorded else torch.zeros
        codes = new((st.B, st.H, need, 2, st.D), dtype=torch.int8, device=st.device)
        scales = new((st.B, st.H, need), dtype=torch.float32, device=st.device)
        if have:
            codes[:, :, :have].copy_(self.codes)
            scales[:, :, :have].copy_(self.scales)
        self.codes, self.scales = codes, scales  # from here on nothing fails
        if other:
            self._store, self.covered, self._recorded = st, 0, None

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
        d = st.descriptor()  # held here while its address is in use
        capture = _lib.calls().block_bounds(ctypes.addressof(d), t0, T, self.block_tokens, self.codes, self.scales)
        if capture:
            self._recorded = (capture, T)
        else:
            self.covered, self._recorded = T, None
        return self

    def bounds(self, first: int = 0) -> torch.Tensor:
        """The key ranges of blocks ``first`` on: fp32 [B, Hkv, n, 2, D],
        lower bounds at index 0 and upper bounds at index 1 of dim 3."""
        n = self.n_blocks - int(first)
        if first < 0 or n < 0 or self.codes is None:
            raise ValueError(f"BlockIndex: first block {first} outside [0, {self.n_blocks}] (or nothing summarised)")
        if self._store is not self.cache.store:
            raise ValueError("BlockIndex: the cache's state was replaced since the last update()")
        return _lib.calls().block_bounds_read(self.codes, self.scales, int(first), n)

    @traced("cq.block_select")
    def select(self, queries: torch.Tensor, top: int, *, first: int = 1, recent: int = 2, starts=None,
               return_scores: bool = False):
        """Up to ``top`` blocks for every query token of ``queries`` [B, Hq,
        Tq, D] (the cache's newest tokens) and kv-head: int32 [B, Hkv, Tq,
        top], ascending, -1 behind.  The ``first`` lowest and ``recent`` highest
        blocks a token may see are always listed, the others by score (ties to
        the lower index).  ``starts``: int64 [B], first real token of each
        sequence.  ``return_scores``: also the listed blocks' scores (fp32, -inf
        behind), by which lists of ranks that share a sequence can be merged.
        Scratch: up to 1 GB of scores at a time, longer chunks go by parts."""
        T = self.cache.offset
        if T == 0 or self.cache.store is not self._store or self.covered != T and self._tokens() != T:
            self.update()
        return _lib.calls().block_select(self.codes, self.scales, self.block_tokens, T, queries, top, first, recent,
                                         starts, return_scores)


@traced("cq.sparse_sdpa")
def chronoquant_sparse_sdpa(queries: torch.Tensor, cache, scale: float, blocks: torch.Tensor, block_tokens: int, *,
                            starts=None, return_lse: bool = False):
    """Attention of ``queries`` [B, Hq, Tq, D] (fp16/bf16, the cache's newest
    tokens) over the tokens of the listed blocks: ``blocks`` int32 [B, Hkv, Tq,
    n], ascending as ``BlockIndex.select`` lists them (an entry that is negative
    or not above its predecessor is left out).  Returns [B, Hq, Tq, D] in the
    query dtype; with ``return_lse`` an fp32 output and the fp32 log-sum-exp [B,
    Hq, Tq] (-inf for a row that sees no token), for merging.

    The layouts of the decode kernel hold queries * scale and the weights times a
    token's value scale in fp16, as it does: ``|queries * scale|`` has to stay
    below 65520 and keeps fp16's digits below 2^-14, and value scales have to stay
    below 256 (residuals of 1792 in 4-bit codes), or a head comes out infinite or
    NaN.  Other layouts keep the query dtype's range.  No gradients: the cache is a
    store of encoded tokens, and the result is detached whatever the queries
    require."""
    st, T = cache.store, cache.offset
    if st is None or T == 0:
        raise ValueError("chronoquant_sparse_sdpa: the cache is empty")
    d = st.descriptor()  # held here while its address is in use
    return _lib.calls().sparse_attention(ctypes.addressof(d), st.buf, T, queries, scale, blocks, block_tokens, starts,
                                         return_lse)
