"""Block index, block selection and sparse attention over the compressed cache.

Every operator is compared with a plain 64-bit implementation on the cache's
own saved state (``cache.state``: the reference layout).

Bars.  Bounds and block lists are whole numbers and fp32 products in a fixed
order: equal.  Attention: the decode kernel rounds P to fp16 (2^-11 relative),
P * scale to fp16, the per-anchor sums of P to fp16 and the denominator is a
sum of the rounded P, so with sum p = 1 the output is within 5 * 2^-11 * max|v|
of the exact one (fp32 score errors of ~1e-5 are inside that), plus half a step
of the output type; the log-sum-exp within 2^-10."""

import ctypes
import math
import threading
import time

import pytest
import torch

from chronoquant_mlx_b200 import (BlockIndex, ChronoQuantCache, _lib, chronoquant_sdpa, chronoquant_sparse_sdpa,
                                  qk_norm_rope)

gpu = pytest.mark.gpu


def make_cache(B, H, T, D, seed=0, dtype=torch.float16, step=None, **kw):
    """A cache of AR(1) keys and values with a few strong key channels."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    k = torch.randn((B, H, T, D), generator=g, device="cuda")
    v = torch.randn((B, H, T, D), generator=g, device="cuda")
    drift = torch.randn((B, H, -(-T // 16), D), generator=g, device="cuda").repeat_interleave(16, 2)[:, :, :T]
    k = 0.35 * k + drift + 2 * torch.randn((1, H, 1, D), generator=g, device="cuda")
    v = 0.3 * v + drift
    cache = ChronoQuantCache(**kw)
    k, v = k.to(dtype), v.to(dtype)
    for a in range(0, T, step or T):
        b = min(T, a + (step or T))
        cache.update_and_fetch(k[:, :, a:b], v[:, :, a:b])
    return cache


def decoded(cache, fp16_keys=False):
    """K and V in 64 bits from the saved state: anchor + code * scale (or the
    keys as reconstruct_history rounds them)."""
    st = cache.state
    kf, packed, scales = [st[0], st[1]], [], []
    rest = st[2:]
    i = 0
    out = []
    T = cache.offset
    for c, s in enumerate((cache.stride_k, cache.stride_v)):
        t = torch.arange(T, device="cuda")
        a = t // s
        x = kf[c][:, :, a].double()
        if T > kf[c].shape[2]:
            pk, sc = rest[i], rest[i + 1]
            i += 2
            w = pk.view(torch.int32).unsqueeze(-1)
            code = (((w >> torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)) & 15) - 8).flatten(-2)
            code = code[..., :x.shape[-1]].double()
            pf = (t - a - 1).clamp(min=0)
            r = (code * sc.double().unsqueeze(-1))[:, :, pf]
            if fp16_keys and c == 0:
                y = (x + r.half().double()).half().double()
            else:
                y = x + r
            x = torch.where((t % s == 0)[:, None], x, y)
        out.append(x)
    return out


def ref_bounds(keys, bt):
    """(codes int [B, H, n, 2, D], scales fp32 [B, H, n]) of fp16-valued keys."""
    B, H, T, D = keys.shape
    lo, hi = [], []
    for a in range(0, T, bt):
        x = keys[:, :, a:a + bt]
        lo.append(torch.where(x.isnan(), math.inf, x).amin(2))
        hi.append(torch.where(x.isnan(), -math.inf, x).amax(2))
    lo, hi = torch.stack(lo, 2), torch.stack(hi, 2)
    none = lo > hi
    lo = torch.where(none, 0.0, lo).clamp(-65504, 65504)
    hi = torch.where(none, 0.0, hi).clamp(-65504, 65504)
    s = (torch.maximum(lo.abs(), hi.abs()).amax(-1).float() / torch.full((), 126.0, device=keys.device)).double()
    d = torch.where(s > 0, s, 1.0).unsqueeze(-1)
    return torch.stack((torch.floor(lo / d), torch.ceil(hi / d)), 3), s.float()


def ref_select(codes, scales, q, T, bt, top, first, recent, starts=None):
    """Lists and scores by the definition, one row at a time."""
    B, Hq, S, D = q.shape
    H = codes.shape[1]
    G = Hq // H
    x = torch.nan_to_num(q.float(), nan=0.0, posinf=65504.0, neginf=-65504.0).clamp(-65504, 65504)
    amax = x.abs().amax(-1, keepdim=True)
    zero = amax < 1e-30
    r = torch.full_like(amax, 127.0) / torch.where(zero, 1.0, amax)
    q8 = torch.where(zero, 0.0, torch.round(x * r)).double().view(B, H, G, S, D)
    sg = torch.where(zero, 0.0, amax / torch.full_like(amax, 127.0)).view(B, H, G, S)
    lists = torch.full((B, H, S, top), -1, dtype=torch.int32)
    out = torch.full((B, H, S, top), -math.inf)
    for b in range(B):
        st = 0 if starts is None else max(0, int(starts[b]))
        for h in range(H):
            dot = (q8[b, h].clamp(min=0) @ codes[b, h, :, 1].T + q8[b, h].clamp(max=0) @ codes[b, h, :, 0].T).float()
            score = (sg[b, h].unsqueeze(-1) * scales[b, h]).float() * dot
            score = score.amax(0).cpu()  # [S, n]
            for i in range(S):
                p = T - S + i
                if st > p:
                    continue
                fb, lb = st // bt, p // bt
                seen = list(range(fb, lb + 1))
                forced = {j for j in seen if j < fb + first or j > lb - recent}
                order = sorted(seen, key=lambda j: (j not in forced, -float(score[i, j]) if j not in forced else 0.0, j))
                got = sorted(order[:top])
                lists[b, h, i, :len(got)] = torch.tensor(got, dtype=torch.int32)
                out[b, h, i, :len(got)] = score[i, got]
    return lists, out


def ref_sparse(K, V, q, scale, blocks, bt, starts=None):
    """64-bit attention over the listed blocks; (out, lse, max|v| per row)."""
    B, Hq, S, D = q.shape
    H, T = K.shape[1], K.shape[2]
    G = Hq // H
    qs = (q * torch.tensor(scale, dtype=q.dtype, device=q.device)).double()
    out = torch.zeros((B, Hq, S, D), dtype=torch.float64, device=q.device)
    lse = torch.full((B, Hq, S), -math.inf, dtype=torch.float64, device=q.device)
    vmax = torch.zeros((B, Hq, S, 1), dtype=torch.float64, device=q.device)
    lists = blocks.cpu()
    for b in range(B):
        st = 0 if starts is None else max(0, int(starts[b]))
        for h in range(H):
            for i in range(S):
                row = lists[b, h, i].tolist()
                keep = [j for n, j in enumerate(row) if j >= 0 and (n == 0 or j > row[n - 1])]
                t = [x for j in keep for x in range(max(st, j * bt), min(T - S + i + 1, (j + 1) * bt))]
                if not t:
                    continue
                t = torch.tensor(t, device=q.device)
                w = qs[b, h * G:(h + 1) * G, i] @ K[b, h, t].T
                lse[b, h * G:(h + 1) * G, i] = torch.logsumexp(w, -1)
                out[b, h * G:(h + 1) * G, i] = torch.softmax(w, -1) @ V[b, h, t]
                vmax[b, h * G:(h + 1) * G, i] = V[b, h, t].abs().max()
    return out, lse, vmax


def check_attention(got, ref, vmax):
    half = torch.finfo(got.dtype).eps / 2
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all()
    tol = 5 * 2.0 ** -11 * vmax + half * ref.abs() + 1e-12
    assert (err <= tol).all(), float((err / tol).max())


def queries(B, Hq, S, D, dtype, seed=5, amp=1.3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (amp * torch.randn((B, Hq, S, D), generator=g, device="cuda")).to(dtype)


# ----------------------------------------------------------------------------- bounds
@gpu
@pytest.mark.parametrize("T,bt", [(1, 16), (15, 16), (64, 64), (65, 64), (333, 64), (700, 128), (1000, 48)])
@pytest.mark.parametrize("kw", [dict(), dict(stride_k=64, stride_v=32, delta_bits_v=3), dict(stride_k=1, stride_v=1),
                                dict(stride_k=12, stride_v=4)])
def test_bounds_equal_definition(T, bt, kw):
    cache = make_cache(2, 3, T, 128, seed=T, **kw)
    index = BlockIndex(cache, bt).update()
    codes, scales = ref_bounds(decoded(cache, fp16_keys=True)[0], bt)
    n = -(-T // bt)
    assert index.n_blocks == n and index.covered == T
    assert torch.equal(index.codes[:, :, :n].double(), codes)
    assert torch.equal(index.scales[:, :, :n], scales)
    assert torch.equal(index.bounds(), codes.float() * scales[..., None, None])
    assert torch.equal(index.bounds(n - 1), (codes.float() * scales[..., None, None])[:, :, n - 1:])
    x = cache.reconstruct_history()[0].double()  # the ranges hold every decoded key
    t = torch.arange(T, device="cuda") // bt
    lo, hi = codes[:, :, :, 0] * scales.double()[..., None], codes[:, :, :, 1] * scales.double()[..., None]
    assert (lo[:, :, t] <= x).all() and (x <= hi[:, :, t]).all()


@gpu
@pytest.mark.parametrize("D", [8, 64, 72, 256])
def test_bounds_head_dims(D):
    cache = make_cache(1, 2, 200, D, seed=D)
    codes, scales = ref_bounds(decoded(cache, fp16_keys=True)[0], 32)
    index = BlockIndex(cache, 32).update()
    assert torch.equal(index.codes[:, :, :7].double(), codes) and torch.equal(index.scales[:, :, :7], scales)


@gpu
def test_bounds_follow_the_cache():
    """Updates after appends of 1 .. 100 tokens (across page and pool growth)
    leave the same ranges as one pass over everything; untouched blocks keep
    their bytes, rows behind the last block stay as they were."""
    g = torch.Generator(device="cuda").manual_seed(2)
    cache = ChronoQuantCache(stride_k=32, stride_v=8)
    index, T = BlockIndex(cache, 64), 0
    for n in (1, 1, 62, 1, 100, 37, 1, 300, 64, 9):
        cache.update_and_fetch(*(torch.randn((2, 2, n, 128), generator=g, device="cuda").half() for _ in range(2)))
        T += n
        index.update()
        assert index.covered == T
        whole = BlockIndex(cache, 64).update()
        m = index.n_blocks
        assert torch.equal(index.codes[:, :, :m], whole.codes[:, :, :m])
        assert torch.equal(index.scales[:, :, :m], whole.scales[:, :, :m])
        assert not index.codes[:, :, m:].any() and not index.scales[:, :, m:].any()
    before = index.codes.clone()
    index.update(T - 1)  # recomputing the last block changes nothing
    assert torch.equal(index.codes, before)
    other = make_cache(2, 2, 100, 128, seed=9)
    cache.state = other.state  # a restored state is another store: the index starts again
    index.update()
    assert index.covered == 100
    assert torch.equal(index.codes[:, :, :2], BlockIndex(other, 64).update().codes[:, :, :2])


@gpu
def test_index_of_a_replaced_state():
    """A cache restored to another state of the same length: ranges of the old
    one are not handed out, and a selection summarises anew."""
    a, b = make_cache(1, 2, 300, 128, seed=1), make_cache(1, 2, 300, 128, seed=2)
    index, q = BlockIndex(a, 32).update(), queries(1, 4, 1, 128, torch.float16)
    index.bounds()
    a.state = b.state
    with pytest.raises(ValueError, match="replaced"):
        index.bounds()
    other = BlockIndex(b, 32)
    assert torch.equal(index.select(q, 5), other.select(q, 5))
    assert torch.equal(index.bounds(), other.bounds())


@gpu
def test_bounds_with_infinite_and_nan_keys():
    """A block with an infinite or NaN anchor keeps finite ranges; the others are untouched."""
    clean, dirty = make_cache(1, 1, 256, 128, seed=4, stride_k=16), make_cache(1, 1, 256, 128, seed=4, stride_k=16)
    st = dirty.state
    st[0][0, 0, 4, 7], st[0][0, 0, 4, 8], st[0][0, 0, 4, 9] = math.nan, math.inf, -math.inf
    dirty.state = st
    a, b = BlockIndex(clean, 64).update(), BlockIndex(dirty, 64).update()
    assert torch.isfinite(b.bounds()).all()
    keep = [0, 2, 3]
    assert torch.equal(a.codes[:, :, keep], b.codes[:, :, keep])
    codes, scales = ref_bounds(decoded(dirty, fp16_keys=True)[0], 64)
    assert torch.equal(b.codes[:, :, :4].double(), codes) and torch.equal(b.scales[:, :, :4], scales)


@gpu
def test_bounds_of_equal_keys_are_exact():
    """All keys zero: zero scale and codes.  One value everywhere: its range is the value."""
    cache = ChronoQuantCache()
    z = torch.zeros((1, 1, 80, 128), device="cuda").half()
    cache.update_and_fetch(z, z)
    index = BlockIndex(cache, 64).update()
    assert not index.bounds().any()


# ----------------------------------------------------------------------------- selection
SELECT = [  # B, H, G, S, T, bt, top, first, recent
    (1, 1, 1, 1, 1, 16, 1, 0, 0), (1, 2, 4, 1, 40, 16, 2, 1, 1), (2, 2, 4, 1, 1000, 32, 8, 1, 2),
    (1, 2, 4, 7, 700, 64, 5, 1, 2), (1, 1, 8, 33, 300, 16, 6, 0, 1), (2, 1, 3, 2, 513, 32, 40, 2, 3),
    (1, 2, 2, 1, 5000, 16, 64, 1, 2), (1, 1, 4, 16, 16, 16, 3, 1, 1), (3, 1, 16, 1, 700, 64, 4, 0, 0),
    (1, 2, 2, 3, 900, 16, 5, 2, 3), (1, 1, 1, 2, 9000, 16, 7, 7, 0), (1, 1, 2, 1, 20000, 16, 300, 1, 2),
    (1, 2, 4, 600, 6000, 16, 20, 1, 2), (1, 1, 32, 2, 3000, 16, 9, 1, 1),
]


@gpu
@pytest.mark.parametrize("shape", SELECT)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_select_equals_definition(shape, dtype):
    B, H, G, S, T, bt, top, first, recent = shape
    cache = make_cache(B, H, T, 128, seed=T + S)
    q = queries(B, H * G, S, 128, dtype)
    index = BlockIndex(cache, bt)
    blocks, scores = index.select(q, top, first=first, recent=recent, return_scores=True)  # updates by itself
    codes, scales = ref_bounds(decoded(cache, fp16_keys=True)[0], bt)
    ref, ref_s = ref_select(codes, scales, q, T, bt, top, first, recent)
    assert torch.equal(blocks.cpu(), ref)
    assert torch.equal(scores.cpu(), ref_s)
    assert torch.equal(index.select(q, top, first=first, recent=recent), blocks)


@gpu
@pytest.mark.parametrize("T,top", [(140000, 64), (140000, 700), (270000, 40), (270000, 3000)])
def test_select_long_rows(T, top):
    """8750 blocks (a row in the registers of 18 warps) and 16875 (the radix
    kernel), with lists shorter and longer than what one warp finishes."""
    cache = make_cache(1, 1, T, 64, seed=T)
    q = queries(1, 2, 1, 64, torch.float16)
    index = BlockIndex(cache, 16).update()
    n = index.n_blocks
    got, s = index.select(q, top, return_scores=True)
    ref, ref_s = ref_select(index.codes[:, :, :n].double(), index.scales[:, :, :n], q, T, 16, top, 1, 2)
    assert torch.equal(got.cpu(), ref) and torch.equal(s.cpu(), ref_s)


@gpu
@pytest.mark.parametrize("blocks", [200, 700, 9000, 17000])
def test_select_many_equal_scores(blocks):
    """Two kinds of block only, more of each than any short list: whole
    classes of equal keys at the threshold, the lowest indexes of them."""
    k = torch.ones((1, 1, blocks * 16, 64), device="cuda").half()
    k.view(1, 1, blocks, 16, 64)[:, :, ::3] = 2
    cache = ChronoQuantCache()
    cache.update_and_fetch(k, k)
    index = BlockIndex(cache, 16)
    q = torch.ones((1, 1, 1, 64), device="cuda").half()
    for top in (10, blocks // 3 + 5, 4000):
        if top > min(4096, blocks):
            continue
        got = index.select(q, top, first=1, recent=2).flatten().tolist()
        order = sorted(range(blocks), key=lambda j: (not (j == 0 or j >= blocks - 2), j % 3 != 0, j))
        assert got == sorted(order[:top])


@gpu
@pytest.mark.parametrize("kind", ["normal", "skewed", "two values", "outliers"])
@pytest.mark.parametrize("S,blocks", [(450, 200), (450, 300), (450, 1000), (100, 1000), (75, 1500), (75, 4000),
                                      (9, 4000), (3, 6000), (40, 9000), (1, 700)])
def test_select_of_many_rows(S, blocks, kind):
    """Every form of the search (a warp, up to four or more warps a row) on
    scores that do and do not look normal, padded and not, for short, middle and
    long lists.  The reference sorts the whole row, equal scores by index."""
    B, H, G, D, bt, first, recent = 2, 4, 2, 64, 16, 1, 2
    T = blocks * bt - 5
    g = torch.Generator(device="cuda").manual_seed(S * blocks)
    k = torch.randn((B, H, blocks, 1, D), generator=g, device="cuda").expand(-1, -1, -1, bt, -1).clone()
    u = torch.rand((B, H, blocks, 1, 1), generator=g, device="cuda")
    if kind == "skewed":
        k *= torch.exp2(-12 * u ** 0.25)
    elif kind == "two values":
        k = torch.ones_like(k) * (1 + (u > 0.6))
    elif kind == "outliers":
        k = torch.where(u > 0.99, 300 * k, k)
    k = k.reshape(B, H, blocks * bt, D)[:, :, :T].half()
    cache = ChronoQuantCache()
    cache.update_and_fetch(k, k)
    index = BlockIndex(cache, bt).update()
    q = queries(B, H * G, S, D, torch.bfloat16, seed=blocks)
    codes, scales = index.codes[:, :, :blocks].double(), index.scales[:, :, :blocks]
    x = q.float()
    amax = x.abs().amax(-1, keepdim=True)
    q8 = torch.round(x * (torch.full_like(amax, 127.0) / amax)).double().view(B, H, G, S, D)
    sg = (amax / torch.full_like(amax, 127.0)).view(B, H, G, S, 1)
    dot = (torch.einsum("bhgsd,bhnd->bhgsn", q8.clamp(min=0), codes[:, :, :, 1])
           + torch.einsum("bhgsd,bhnd->bhgsn", q8.clamp(max=0), codes[:, :, :, 0])).float()
    score = ((sg * scales[:, :, None, None]) * dot).amax(2)  # [B, H, S, n]
    j = torch.arange(blocks, device="cuda")
    p = (T - S + torch.arange(S, device="cuda")).view(1, 1, S, 1)
    for starts in (None, torch.tensor([37, T // 3], device="cuda")):
        st = torch.zeros((B, 1, 1, 1), dtype=torch.int64, device="cuda") if starts is None else starts.view(B, 1, 1, 1)
        fb, lb = st // bt, p // bt
        seen = (j >= fb) & (j <= lb)
        forced = seen & ((j < fb + first) | (j > lb - recent))
        rank = torch.where(forced, math.inf, torch.where(seen, score, -math.inf))
        order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
        for top in (4, 40, 100, min(blocks, 900)):
            want = torch.where(seen.expand_as(rank).gather(-1, order[..., :top]), order[..., :top], blocks)
            want = want.sort(-1).values
            want_s = torch.where(want < blocks, score.gather(-1, want.clamp(max=blocks - 1)), -math.inf)
            got, s = index.select(q, top, first=first, recent=recent, starts=starts, return_scores=True)
            assert torch.equal(got, torch.where(want < blocks, want, -1).int()), top
            assert torch.equal(s, want_s), top


@gpu
@pytest.mark.parametrize("D", [8, 32, 64, 72, 96, 256])
def test_select_head_dims(D):
    cache = make_cache(2, 2, 600, D, seed=D)
    q = queries(2, 6, 3, D, torch.float16)
    got = BlockIndex(cache, 16).select(q, 9)
    codes, scales = ref_bounds(decoded(cache, fp16_keys=True)[0], 16)
    assert torch.equal(got.cpu(), ref_select(codes, scales, q, 600, 16, 9, 1, 2)[0])


@gpu
def test_select_ties_go_to_the_lowest_index():
    """Constant keys: every block has the same score, so the list is the first
    ones and the recent ones; a zero query scores every block 0."""
    cache = ChronoQuantCache()
    one = torch.ones((1, 1, 640, 128), device="cuda").half()
    cache.update_and_fetch(one, one)
    index = BlockIndex(cache, 16)
    for q in (queries(1, 4, 1, 128, torch.float16), torch.zeros((1, 4, 1, 128), device="cuda").half()):
        got, s = index.select(q, 10, first=1, recent=2, return_scores=True)
        assert got.flatten().tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 38, 39]
        assert (s == s.flatten()[0]).all()


@gpu
def test_select_odd_queries():
    """NaN, infinite, huge, tiny and denormal query values follow the definition; strided queries too."""
    cache = make_cache(1, 2, 900, 128, seed=1)
    index = BlockIndex(cache, 16).update()
    codes, scales = ref_bounds(decoded(cache, fp16_keys=True)[0], 16)
    q = queries(1, 8, 4, 128, torch.bfloat16)
    q[0, 0, 0, 3], q[0, 1, 0, 4], q[0, 2, 1, 5] = math.nan, math.inf, -math.inf
    q[0, 3, 2] *= 1e36
    q[0, 4, 2] *= 1e-36
    q[0, 5, 3] = 0
    q[0, 4:8, 3] = 1e-39
    ref, ref_s = ref_select(codes, scales, q, 900, 16, 12, 1, 2)
    got, s = index.select(q, 12, return_scores=True)
    assert torch.equal(got.cpu(), ref) and torch.equal(s.cpu(), ref_s)
    strided = torch.zeros((1, 4, 8, 256), dtype=torch.bfloat16, device="cuda").transpose(1, 2)[..., 64:192]
    strided.copy_(q)
    assert torch.equal(index.select(strided, 12), got)
    spread = torch.zeros((1, 8, 4, 256), dtype=torch.bfloat16, device="cuda")[..., ::2]
    spread.copy_(q)
    assert torch.equal(index.select(spread, 12), got)


@gpu
def test_select_padded_batch():
    """Left padding: nothing before a sequence's first token is listed; a
    sequence that is all padding gets an empty list, a negative start is 0."""
    cache = make_cache(5, 1, 500, 128, seed=6)
    starts = torch.tensor([0, 130, 499, 500, -3], device="cuda")
    q = queries(5, 4, 3, 128, torch.bfloat16)
    index = BlockIndex(cache, 16).update()
    codes, scales = ref_bounds(decoded(cache, fp16_keys=True)[0], 16)
    got, s = index.select(q, 8, starts=starts, return_scores=True)
    ref, ref_s = ref_select(codes, scales, q, 500, 16, 8, 1, 2, starts)
    assert torch.equal(got.cpu(), ref) and torch.equal(s.cpu(), ref_s)
    assert (got[3] == -1).all() and (got[2, 0, 0] == -1).all() and got[2, 0, 2, 0] == 31


# ----------------------------------------------------------------------------- attention
LAYOUTS = [dict(), dict(stride_k=64, stride_v=32, delta_bits_v=3), dict(stride_k=16, stride_v=16),
           dict(stride_k=64, stride_v=32, delta_bits_v=3, v_pack=3), dict(stride_k=32, stride_v=8, delta_bits_v=2,
                                                                          v_pack=2),
           dict(stride_k=12, stride_v=4), dict(stride_k=1, stride_v=1)]
SPARSE = [  # B, H, G, S, T, bt, top
    (1, 1, 1, 1, 1, 64, 1), (2, 2, 4, 1, 333, 64, 3), (1, 2, 8, 1, 2000, 64, 9), (1, 2, 4, 5, 700, 64, 4),
    (1, 1, 16, 2, 400, 128, 3), (2, 1, 3, 40, 257, 16, 5), (1, 2, 2, 1, 1500, 256, 4), (2, 1, 7, 3, 130, 48, 6),
    (2, 2, 1, 21, 900, 64, 4), (1, 2, 2, 10, 1300, 64, 6), (1, 2, 3, 9, 1300, 64, 5), (1, 1, 4, 70, 1000, 64, 3),
    (1, 1, 4, 2, 800, 64, 300),
]


@gpu
@pytest.mark.parametrize("kw", LAYOUTS)
@pytest.mark.parametrize("shape", SPARSE)
def test_sparse_attention_matches_64_bits(kw, shape):
    B, H, G, S, T, bt, top = shape
    cache = make_cache(B, H, T, 128, seed=T, **kw)
    dtype = torch.bfloat16 if T % 2 else torch.float16
    q = queries(B, H * G, S, 128, dtype)
    blocks = BlockIndex(cache, bt).select(q, top, first=0, recent=1)
    scale = 128 ** -0.5
    ref, rlse, vmax = ref_sparse(*decoded(cache), q, scale, blocks, bt)
    check_attention(chronoquant_sparse_sdpa(q, cache, scale, blocks, bt), ref, vmax)
    out, lse = chronoquant_sparse_sdpa(q, cache, scale, blocks, bt, return_lse=True)
    assert out.dtype == lse.dtype == torch.float32
    check_attention(out, ref, vmax)
    assert (lse.double() - rlse).abs().max() <= 2.0 ** -10


@gpu
@pytest.mark.parametrize("D", [8, 64, 72, 256])
def test_sparse_attention_head_dims(D):
    cache = make_cache(2, 2, 300, D, seed=D)
    q = queries(2, 4, 2, D, torch.float16)
    blocks = BlockIndex(cache, 32).select(q, 4)
    ref, _, vmax = ref_sparse(*decoded(cache), q, D ** -0.5, blocks, 32)
    check_attention(chronoquant_sparse_sdpa(q, cache, D ** -0.5, blocks, 32), ref, vmax)


@gpu
@pytest.mark.parametrize("kw", LAYOUTS[:3] + LAYOUTS[5:6])
def test_sparse_attention_over_every_block_is_dense_attention(kw):
    """With every block listed the result is the dense decode's, and lists that
    split the blocks merge back by their log-sum-exps."""
    cache = make_cache(2, 2, 777, 128, seed=3, **kw)
    q = queries(2, 8, 1, 128, torch.float16)
    scale = 128 ** -0.5
    every = torch.arange(13, dtype=torch.int32, device="cuda").expand(2, 2, 1, 13)
    K, V = decoded(cache)
    ref, _, vmax = ref_sparse(K, V, q, scale, every, 64)
    check_attention(chronoquant_sparse_sdpa(q, cache, scale, every, 64), ref, vmax)
    check_attention(chronoquant_sdpa(q, None, None, cache, scale), ref, vmax)
    parts = [chronoquant_sparse_sdpa(q, cache, scale, every[..., s], 64, return_lse=True)
             for s in (slice(0, 5), slice(5, 6), slice(6, 13))]
    lse = torch.stack([p[1] for p in parts])
    w = torch.softmax(lse, 0).unsqueeze(-1)
    check_attention((w * torch.stack([p[0] for p in parts])).sum(0), ref, vmax)


@gpu
@pytest.mark.parametrize("kw", [LAYOUTS[0], LAYOUTS[1], LAYOUTS[5]])
def test_sparse_attention_lists(kw):
    """Absent entries anywhere, repeats, blocks behind the query or past the
    cache, an empty list (zeros, -inf) and lists of one entry."""
    cache = make_cache(1, 3, 500, 128, seed=8, **kw)
    q = queries(1, 6, 2, 128, torch.float16)
    rows = [[[-1, 0, 0, 3, 7, 7], [2, -1, -1, 5, 6, 7]], [[-1] * 6, [7, 8, 100, 2 ** 30, 2 ** 31 - 1, -7]],
            [[7, -1, -1, -1, -1, -1], [8, 9, 10, 11, 12, 13]]]
    blocks = torch.tensor(rows, dtype=torch.int32, device="cuda").unsqueeze(0)
    ref, rlse, vmax = ref_sparse(*decoded(cache), q, 0.1, blocks, 64)
    out, lse = chronoquant_sparse_sdpa(q, cache, 0.1, blocks, 64, return_lse=True)
    check_attention(out, ref, vmax)
    empty = torch.isinf(rlse)
    assert torch.equal(torch.isinf(lse), empty) and empty[0, 2, 0] and empty[0, 5, 1]
    assert not out[empty].any()
    assert (lse[~empty].double() - rlse[~empty]).abs().max() <= 2.0 ** -10
    one = blocks[..., 3:4]
    ref, _, vmax = ref_sparse(*decoded(cache), q, 0.1, one, 64)
    check_attention(chronoquant_sparse_sdpa(q, cache, 0.1, one, 64), ref, vmax)  # a strided list


@gpu
@pytest.mark.parametrize("kw", [LAYOUTS[0], LAYOUTS[1], LAYOUTS[5]])
def test_sparse_attention_padded_batch(kw):
    """Left padding that ends inside a block, at a block border, in the last
    token and beyond it (zeros); NaN in the padding reaches no output."""
    T = 300
    g = torch.Generator(device="cuda").manual_seed(1)
    starts = torch.tensor([0, 70, 128, 299, 300, -5], device="cuda")
    k, v = (torch.randn((6, 2, T, 128), generator=g, device="cuda").half() for _ in range(2))
    for b, s in enumerate(starts.tolist()):
        if 0 < s <= T:  # the codec spreads an anchor over its stride: poison whole anchor groups only
            s = s // 64 * 64
            k[b, :, :s], v[b, :, :s] = math.nan, math.nan
    cache = ChronoQuantCache(**kw)
    if 64 % cache.stride_k or 64 % cache.stride_v:
        k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    cache.update_and_fetch(k, v)
    q = queries(6, 8, 2, 128, torch.bfloat16)
    index = BlockIndex(cache, 16 if kw == LAYOUTS[5] else 64)
    blocks = index.select(q, 3, starts=starts)
    K, V = decoded(cache)
    ref, _, vmax = ref_sparse(K, V, q, 0.09, blocks, index.block_tokens, starts)
    out = chronoquant_sparse_sdpa(q, cache, 0.09, blocks, index.block_tokens, starts=starts)
    check_attention(out, ref, vmax)
    assert not out[4].any() and not out[3, :, 0].any() and out[3, :, 1].any()


@gpu
@pytest.mark.parametrize("kw", [LAYOUTS[0], LAYOUTS[1], LAYOUTS[2], LAYOUTS[4], LAYOUTS[5]])
@pytest.mark.parametrize("G", [1, 2, 4, 8])
def test_infinite_values_stay_with_the_queries_that_see_them(kw, G):
    """Query tokens that are computed together: a NaN or infinite value in a
    block that only one of them lists, and in the newest token, which only the
    last one sees, reaches that one's output and no other's."""
    T, S = 500, 6
    cache = make_cache(1, 1, T, 128, seed=3, **kw)
    st = cache.state
    st[1][0, 0, 64 // cache.stride_v, 5] = math.nan  # the V anchor of token 64: block 1
    st[1][0, 0, 192 // cache.stride_v, 9] = math.inf  # of token 192: block 3
    clean = ChronoQuantCache(**kw)
    clean.state = [x.clone() for x in cache.state]
    cache.state = st
    q = queries(1, G, S, 128, torch.float16)
    rows = [[0, 2, 7], [0, 1, 7], [2, 3, 7], [4, 5, 7], [0, 3, 7], [2, 4, 7]]
    blocks = torch.tensor(rows, dtype=torch.int32, device="cuda").view(1, 1, S, 3)
    got = chronoquant_sparse_sdpa(q, cache, 0.1, blocks, 64)
    want = chronoquant_sparse_sdpa(q, clean, 0.1, blocks, 64)
    for i, hit in enumerate((None, 5, 9, None, 9, None)):
        if hit is None:
            assert torch.equal(got[:, :, i], want[:, :, i])
        else:
            assert not torch.isfinite(got[0, :, i, hit]).any()
    # the newest token: an I-frame at 448 with an infinite channel, seen by the last of 3 queries
    short = ChronoQuantCache(**kw)
    k, v = (torch.randn((1, 1, 449, 128), device="cuda").half() for _ in range(2))
    if 448 % cache.stride_v == 0:
        v[..., 448, 3] = math.inf
        short.update_and_fetch(k, v)
        qs, row = queries(1, G, 3, 128, torch.float16), torch.tensor([0, 3, 6, 7], dtype=torch.int32, device="cuda")
        out = chronoquant_sparse_sdpa(qs, short, 0.1, row.expand(1, 1, 3, 4), 64)
        assert torch.isfinite(out[:, :, :2]).all() and not torch.isfinite(out[0, :, 2, 3]).any()


def score_slack(cache, q, scale):
    """How far scores may be off, beside the roundings that check_attention
    counts.  q.code is accumulated over nibbles n <= 15 from -8 sum q on, so
    partial sums stay below 24 * sum|q|; each of at most 16 accumulation steps
    errs by 2^-23 of them, and the token's scale multiplies the result.  The
    anchor's product errs by 16 * 2^-23 * sum|q| * max|anchor|."""
    st = cache.state
    qsum = (q * torch.tensor(scale, dtype=q.dtype, device="cuda")).double().abs().sum(-1).max()
    return 16 * 2.0 ** -23 * qsum * (24 * st[3].double().max() + st[0].double().abs().max())


@gpu
def test_sparse_attention_extreme_scores():
    """Scores of some thousands: no overflow, and few keys decide."""
    cache = make_cache(1, 1, 400, 128, seed=2)
    q = queries(1, 4, 1, 128, torch.float16, amp=300.0)
    blocks = torch.tensor([0, 2, 4, 6], dtype=torch.int32, device="cuda").view(1, 1, 1, 4)
    K, V = decoded(cache)
    ref, rlse, vmax = ref_sparse(K, V, q, 0.25, blocks, 64)
    out, lse = chronoquant_sparse_sdpa(q, cache, 0.25, blocks, 64, return_lse=True)
    slack = score_slack(cache, q, 0.25)
    assert (lse.double() - rlse).abs().max() <= 2.0 ** -10 + slack
    assert ((out.double() - ref).abs() <= (5 * 2.0 ** -11 + 2 * slack) * vmax).all()


@gpu
@pytest.mark.parametrize("kw", [LAYOUTS[0], LAYOUTS[1]])
def test_sparse_attention_tiny_queries_of_large_keys(kw):
    """Query values that are subnormal in fp16 against keys of thousands: the
    scores are sums of products of subnormal numbers."""
    g = torch.Generator(device="cuda").manual_seed(8)
    k = (3000 * torch.randn((1, 1, 400, 128), generator=g, device="cuda")).half()
    v = torch.randn((1, 1, 400, 128), generator=g, device="cuda").half()
    cache = ChronoQuantCache(**kw)
    cache.update_and_fetch(k, v)
    q = queries(1, 4, 2, 128, torch.float16, amp=2.0 ** -13)
    blocks = torch.tensor([0, 1, 4, 6], dtype=torch.int32, device="cuda").expand(1, 1, 2, 4)
    K, V = decoded(cache)
    ref, rlse, vmax = ref_sparse(K, V, q, 0.25, blocks, 64)
    assert rlse.max() > math.log(3 * 64 + 16) + 0.2  # 208 tokens, and their scores count
    out, lse = chronoquant_sparse_sdpa(q, cache, 0.25, blocks, 64, return_lse=True)
    slack = score_slack(cache, q, 0.25)
    assert (lse.double() - rlse).abs().max() <= 2.0 ** -10 + slack
    assert ((out.double() - ref).abs() <= (5 * 2.0 ** -11 + 2 * slack) * vmax).all()


@gpu
def test_run_of_the_operators_together():
    """A decode loop as a program runs it: append, update, select, attend --
    the whole against 64 bits at every step, across block and page ends."""
    g = torch.Generator(device="cuda").manual_seed(11)
    cache = make_cache(2, 2, 250, 128, seed=1, stride_k=64, stride_v=32, delta_bits_v=3)
    index = BlockIndex(cache, 64).update()
    for step in range(10):
        cache.update_and_fetch(*(torch.randn((2, 2, 1, 128), generator=g, device="cuda").bfloat16() for _ in range(2)))
        q = queries(2, 8, 1, 128, torch.bfloat16, seed=step)
        index.update()
        blocks = index.select(q, 3, first=1, recent=1)
        codes, scales = ref_bounds(decoded(cache, fp16_keys=True)[0], 64)
        assert torch.equal(blocks.cpu(), ref_select(codes, scales, q, cache.offset, 64, 3, 1, 1)[0])
        out = chronoquant_sparse_sdpa(q, cache, 128 ** -0.5, blocks, 64)
        ref, _, vmax = ref_sparse(*decoded(cache), q, 128 ** -0.5, blocks, 64)
        check_attention(out, ref, vmax)


@gpu
def test_captured_and_on_another_stream():
    """The three calls captured into one graph and replayed with other queries,
    and two captures replayed in turn on a side stream: their own results."""
    cache = make_cache(1, 2, 900, 128, seed=5)
    index = BlockIndex(cache, 32).update()
    qa, qb = queries(1, 8, 1, 128, torch.bfloat16, seed=1), queries(1, 8, 1, 128, torch.bfloat16, seed=2)

    def step(q):
        blocks = index.update(cache.offset - 1).select(q, 7)
        return blocks, chronoquant_sparse_sdpa(q, cache, 0.1, blocks, 32)

    want = [[x.clone() for x in step(q)] for q in (qa, qb)]
    bufs, graphs = [torch.empty_like(qa), torch.empty_like(qa)], []
    for q in bufs:
        q.copy_(qa)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(q)
        graphs.append((graph, out))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        bufs[0].copy_(qa)
        bufs[1].copy_(qb)
        for _ in range(3):
            for graph, _ in graphs:
                graph.replay()
        bufs[0].copy_(qb)
        graphs[0][0].replay()
        got0 = [x.clone() for x in graphs[0][1]]
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(got0, want[1]):
        assert torch.equal(x, y)
    for x, y in zip(graphs[1][1], want[1]):
        assert torch.equal(x, y)


# ----------------------------------------------------------------------------- refusals
@gpu
def test_refusals():
    cache = make_cache(2, 2, 100, 128)
    index = BlockIndex(cache, 32).update()
    q = queries(2, 4, 1, 128, torch.float16)
    blocks = index.select(q, 3)
    for kw in (dict(top=0), dict(top=2, first=1, recent=2), dict(top=5000), dict(top=3, first=-1)):
        with pytest.raises(ValueError):
            index.select(q, **kw)
    bad = [q[:1], q[:, :3], q[..., :64], q[0], q.expand(2, 4, 101, 128), q[:, :0], q[:, :, :0]]
    for x in bad:
        with pytest.raises(ValueError):
            index.select(x, 3)
        with pytest.raises(ValueError):
            chronoquant_sparse_sdpa(x, cache, 1.0, blocks, 32)
    with pytest.raises(TypeError):
        index.select(q.float(), 3)
    with pytest.raises(TypeError):
        chronoquant_sparse_sdpa(q.float(), cache, 1.0, blocks, 32)
    with pytest.raises(ValueError):
        index.select(q.cpu(), 3)
    for x in (blocks.long(), blocks[0], blocks[:1], blocks[..., :0], blocks.cpu(), blocks.expand(2, 2, 2, 3)):
        with pytest.raises(ValueError):
            chronoquant_sparse_sdpa(q, cache, 1.0, x, 32)
    for s in (torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"),
              torch.zeros(2, dtype=torch.int64)):
        with pytest.raises(ValueError):
            index.select(q, 3, starts=s)
        with pytest.raises(ValueError):
            chronoquant_sparse_sdpa(q, cache, 1.0, blocks, 32, starts=s)
    for bt in (0, 8, 40):
        with pytest.raises(ValueError):
            chronoquant_sparse_sdpa(q, cache, 1.0, blocks, bt)
    with pytest.raises(ValueError):
        index.update(101)
    with pytest.raises(ValueError):
        index.bounds(5)
    with pytest.raises(ValueError):
        index.bounds(-1)


def test_empty_cache_and_bad_blocks_are_refused():
    cache = ChronoQuantCache()
    for bt in (0, 8, 17, -64):
        with pytest.raises(ValueError):
            BlockIndex(cache, bt)
    index = BlockIndex(cache)
    with pytest.raises(ValueError, match="empty"):
        index.update()
    with pytest.raises(ValueError):
        index.bounds()
    with pytest.raises(ValueError, match="empty"):
        index.select(torch.zeros((1, 1, 1, 128), dtype=torch.float16), 3)
    with pytest.raises(ValueError, match="empty"):
        chronoquant_sparse_sdpa(torch.zeros((1, 1, 1, 128)), cache, 1.0, torch.zeros((1, 1, 1, 1)), 64)
    assert index.n_blocks == 0 and index.nbytes == 0


def _desc(**over):
    d = _lib.CqPagedCache()
    d.batch, d.kv_heads, d.head_dim, d.page_tokens, d.max_pages, d.n_pages = 2, 8, 128, 256, 4, 8
    d.block_table = 0x1000
    for name, s in (("k", 32), ("v", 8)):
        c = getattr(d, name)
        c.stride, c.bits, c.anchors_per_page, c.pframes_per_page = s, 4, 256 // s, 256 - 256 // s
        c.scale_row, c.scale_index = 256, 1
        c.keyframes, c.codes, c.scales = 0x2000, 0x3000, 0x4000
    for k, v in over.items():
        setattr(d, k, v)
    return d


P = 0x10000  # a pointer that the refused calls never follow
BOUNDS = dict(t0=0, T=1000, bt=64, codes=P, scales=P, max_blocks=16)
SELECT_ARGS = dict(codes=P, scales=P, max_blocks=16, bt=64, B=2, H=8, D=72, T=1000, len=None, q=P, dt=0, Hq=32, S=1,
                   sb=4096, sh=128, sq=128, starts=None, first=1, recent=2, top=8, blocks=P, scores=None, ws=P,
                   nws=1 << 20)
SPARSE_ARGS = dict(T=1000, len=None, q=P, dt=0, Hq=32, S=1, sb=4096, sh=128, sq=128, scale=1.0, starts=None, blocks=P,
                   top=8, bt=64, out=P, odt=0, lse=None, ws=P, nws=1 << 30)


@pytest.mark.parametrize("over,status", [
    (dict(codes=None), -1), (dict(scales=None), -1), (dict(bt=0), -1), (dict(T=0), -1), (dict(T=1025), -1),
    (dict(max_blocks=15), -1), (dict(t0=-1), -1), (dict(t0=1001), -1)])
def test_c_bounds_refusals(over, status):
    a = {**BOUNDS, **over}
    d = ctypes.byref(_desc())
    assert _lib.lib().cq_block_bounds(d, *a.values(), None) == status
    assert _lib.lib().cq_last_error()
    if "t0" not in over:
        assert _lib.lib().cq_block_bounds_at(d, P, a["T"], 1, a["bt"], a["codes"], a["scales"], a["max_blocks"],
                                             None) == status


@pytest.mark.parametrize("over,status", [
    (dict(codes=None), -1), (dict(q=None), -1), (dict(blocks=None), -1), (dict(dt=2), -2), (dict(D=12), -2),
    (dict(D=264), -2), (dict(Hq=12), -1), (dict(Hq=0), -1), (dict(S=0), -1), (dict(S=1001), -1), (dict(top=0), -1),
    (dict(top=2), -1), (dict(first=-1), -1), (dict(recent=-1), -1), (dict(top=4097), -2), (dict(max_blocks=15), -1),
    (dict(ws=None), -4), (dict(nws=8), -4), (dict(bt=0), -1), (dict(B=0), -1), (dict(recent=2 ** 31 - 1), -1),
    (dict(codes=P + 8), -1), (dict(ws=P + 4), -1)])
def test_c_select_refusals(over, status):
    assert _lib.lib().cq_block_select(*{**SELECT_ARGS, **over}.values(), None) == status


@pytest.mark.parametrize("over,status", [
    (dict(q=None), -1), (dict(blocks=None), -1), (dict(out=None), -1), (dict(dt=2), -2), (dict(odt=3), -2),
    (dict(Hq=12), -1), (dict(S=0), -1), (dict(S=1001), -1), (dict(T=1025), -1), (dict(top=0), -1), (dict(bt=0), -1),
    (dict(top=4097), -2), (dict(ws=None), -4), (dict(nws=64), -4)])
def test_c_sparse_refusals(over, status):
    assert _lib.lib().cq_sparse_attention(ctypes.byref(_desc()), *{**SPARSE_ARGS, **over}.values(), None) == status


def test_c_bounds_read_refusals():
    L = _lib.lib()
    for args in ((None, P, 16, 16, 0, 4, 128, P), (P, P, 16, 16, 0, 17, 128, P), (P, P, 16, 16, -1, 4, 128, P),
                 (P, P, 16, 16, 13, 4, 128, P), (P, P, 0, 16, 0, 4, 128, P), (P, P, 16, 16, 0, 4, 300, P),
                 (P, P, 16, 16, 0, 4, 128, None)):
        assert L.cq_block_bounds_read(*args, None) == -1


def test_c_sizes_past_32_bits_are_refused():
    L, n, big = _lib.lib(), ctypes.c_size_t(), 2 ** 31 - 1
    far = ctypes.byref(_desc(max_pages=big))  # maps 2^39 tokens
    for T in (2 ** 62, 2 ** 63 - 1):  # sums with a page's or a block's tokens would wrap
        assert L.cq_block_bounds(far, 0, T, 64, P, P, 2 ** 40, None) == -1
        assert L.cq_block_bounds_at(far, P, T, 1, 64, P, P, 2 ** 40, None) == -1
        assert L.cq_block_select(*{**SELECT_ARGS, "T": T, "max_blocks": 2 ** 62}.values(), None) == -1
        assert L.cq_sparse_attention(far, *{**SPARSE_ARGS, "T": T}.values(), None) == -1
    assert L.cq_block_bounds(far, 0, 2 ** 39 - 256, 64, P, P, 2 ** 40, None) == -2  # 2^33 blocks
    # groups of 2^30 heads and more, and rows past 2^31
    assert L.cq_block_select_workspace(1, 1, 128, big, 1, 64, 64, ctypes.byref(n)) == 0 and n.value
    assert L.cq_block_select_workspace(big, big, 128, big, 1, 64, 64, ctypes.byref(n)) == -2
    assert L.cq_block_select_workspace(1, 2, 128, 2, 2 ** 30, 2 ** 31, 64, ctypes.byref(n)) == -2
    for over in (dict(Hq=2 ** 30), dict(S=2 ** 28, T=2 ** 29)):
        assert L.cq_sparse_attention(far, *{**SPARSE_ARGS, **over}.values(), None) == -2
    assert L.cq_block_bounds_read(P, P, 2 ** 40, 2 ** 40, 0, 2 ** 40, 128, P, None) == -1


@gpu
def test_a_captured_update_counts_once_it_has_run():
    """update() in a capture summarises nothing until the graph is replayed:
    what runs meanwhile does not take the ranges for granted."""
    cache = make_cache(2, 2, 150, 128, seed=3)
    index = BlockIndex(cache, 32)
    index.reserve(400)
    index.update()
    more = make_cache(2, 2, 100, 128, seed=4).reconstruct_history()
    cache.update_and_fetch(*more)
    q = queries(2, 8, 1, 128, torch.float16)
    fresh = BlockIndex(cache, 32).update()
    want, bounds = fresh.select(q, 4, return_scores=True), fresh.bounds()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        ranges = index.update().bounds()  # 250 tokens here, recorded
        lists = index.select(q, 4)
        assert index.n_blocks == 8
    assert index.covered == 150 and index.n_blocks == 5 and index.bounds().shape[2] == 5
    with torch.cuda.graph(second):
        others = index.select(q, 4, return_scores=True)  # its own update, not the other graph's
    second.replay()
    assert torch.equal(others[0], want[0]) and torch.equal(others[1], want[1])
    index.codes[:, :, 4:].zero_()  # as before the replay
    got = index.select(q, 4, return_scores=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert index.covered == 250 and torch.equal(index.bounds(), bounds)
    index.codes[:, :, 4:].zero_()
    first.replay()
    assert torch.equal(ranges, bounds) and torch.equal(lists, want[0])
    assert torch.equal(index.bounds(), bounds)


@gpu
def test_an_index_allocated_in_a_capture():
    """An index made inside a capture computes everything when replayed.  A
    replay summarises the tokens of the capture, so of what other calls computed
    meanwhile its last block alone is lost, which an update from there brings back."""
    cache = make_cache(1, 2, 200, 128, seed=3)
    q = queries(1, 8, 1, 128, torch.float16)
    want = BlockIndex(cache, 32).select(q, 3)
    index, graph = BlockIndex(cache, 32), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = index.update().select(q, 3)
    graph.replay()
    assert torch.equal(got, want)
    cache.update_and_fetch(*(x[:, :, :30] for x in make_cache(1, 2, 100, 128, seed=4).reconstruct_history()))
    index.update()
    graph.replay()
    now = BlockIndex(cache, 32).update().bounds()
    assert torch.equal(index.bounds()[:, :, :6], now[:, :, :6]) and torch.equal(index.bounds(7), now[:, :, 7:])
    assert torch.equal(index.update(200).bounds(), now)


@gpu
def test_an_index_does_not_grow_in_a_capture():
    """Growing moves the ranges; a replay would copy them from memory given
    back since.  Refused, and the index still works."""
    cache = make_cache(1, 1, 250, 128, seed=3)
    index = BlockIndex(cache, 32).update()
    cache.update_and_fetch(*make_cache(1, 1, 600, 128, seed=4).reconstruct_history())  # the pool grows
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="reserve"):
        with torch.cuda.graph(graph):
            index.bounds()  # (a graph of something)
            index.update()
    assert index.covered == 250
    assert torch.equal(index.update().bounds(), BlockIndex(cache, 32).update().bounds())


@gpu
def test_an_index_without_memory_to_grow_is_left_as_it_was(monkeypatch):
    """No memory for the ranges of a restored or longer cache: the call fails,
    and the next one starts over."""
    cache = make_cache(1, 1, 100, 128, seed=3)
    index = BlockIndex(cache, 32).update()
    q = queries(1, 4, 1, 128, torch.float16)
    zeros = torch.zeros

    def refuse(size, **kw):
        if kw.get("dtype") is torch.float32:  # the second of the index's two tensors
            raise torch.cuda.OutOfMemoryError("no memory")
        return zeros(size, **kw)

    for other in (make_cache(1, 1, 700, 128, seed=5), make_cache(1, 1, 90, 128, seed=6)):
        cache.state = other.state
        with monkeypatch.context() as m:
            m.setattr(torch, "zeros", refuse)
            for call in (index.update, lambda: index.select(q, 3), index.update):
                with pytest.raises(torch.cuda.OutOfMemoryError):
                    call()
            with pytest.raises(ValueError, match="replaced"):
                index.bounds()
        assert torch.equal(index.select(q, 3), BlockIndex(other, 32).select(q, 3))
        assert torch.equal(index.bounds(), BlockIndex(other, 32).update().bounds())


@gpu
def test_other_threads_run_while_a_call_waits():
    """A call that waits for room in the launch queue holds no other Python
    thread up: this one keeps waking every millisecond or so meanwhile."""
    cache = make_cache(1, 1, 500, 128)
    index = BlockIndex(cache, 32).update()
    q = queries(1, 4, 1, 128, torch.float16)
    qkv, f = torch.zeros((1, 1, 384), device="cuda"), torch.ones(64, device="cuda")
    pos = torch.zeros(1, dtype=torch.int64, device="cuda")
    blocks = index.select(q, 3)
    calls = {"update": lambda: index.update(499), "bounds": index.bounds, "select": lambda: index.select(q, 3),
             "attention": lambda: chronoquant_sparse_sdpa(q, cache, 0.1, blocks, 32),
             "rotation": lambda: qk_norm_rope(qkv, 1, 1, f, pos)}
    for name, call in calls.items():
        call()
        torch.cuda.synchronize()
        done = threading.Event()

        def work():
            for _ in range(3000):  # the queue holds about a thousand launches
                call()
            done.set()

        torch.cuda._sleep(1_200_000_000)  # cycles: 0.6 s
        thread = threading.Thread(target=work)
        worst, last = 0.0, time.perf_counter()
        thread.start()
        while not done.is_set():
            time.sleep(0.001)
            now = time.perf_counter()
            worst, last = max(worst, now - last), now
        thread.join()
        torch.cuda.synchronize()
        assert worst < 0.3, (name, worst)


@gpu
@pytest.mark.parametrize("padded", [False, True])
def test_select_of_very_many_scores_bounds_its_memory(padded):
    """A chunk of queries over many blocks (a third more scores than 1 GB
    holds): listed by parts of the chunk, as one call lists them."""
    B, H, G, S, D, bt, top, first, recent = 2, 4, 2, 3000, 64, 16, 12, 1, 2
    T = 240000 - 3
    n = -(-T // bt)
    cache = make_cache(B, H, T, D, seed=9)
    index = BlockIndex(cache, bt).update()
    q = queries(B, H * G, S, D, torch.bfloat16)
    starts = torch.tensor([3, T - S + 700], device="cuda") if padded else None
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got, s = index.select(q, top, first=first, recent=recent, starts=starts, return_scores=True)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < 1100 << 20
    codes, scales = index.codes[:, :, :n].double(), index.scales[:, :, :n]
    j = torch.arange(n, device="cuda")
    lb = (T - S + torch.arange(S, device="cuda"))[:, None] // bt
    for b in range(B):
        st = 0 if starts is None else int(starts[b])
        fb = st // bt
        x = q[b].float().view(H, G, S, D)
        amax = x.abs().amax(-1, keepdim=True)
        q8 = torch.round(x * (torch.full_like(amax, 127.0) / amax)).double()
        sg = amax / torch.full_like(amax, 127.0)
        for h in range(H):
            dot = (q8[h].clamp(min=0) @ codes[b, h, :, 1].T + q8[h].clamp(max=0) @ codes[b, h, :, 0].T).float()
            score = ((sg[h] * scales[b, h]) * dot).amax(0)
            seen = (j >= fb) & (j <= lb) & (torch.arange(S, device="cuda")[:, None] + T - S >= st)
            rank = torch.where((j < fb + first) | (j > lb - recent), math.inf, score)
            rank = torch.where(seen, rank, -math.inf)
            order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :top]
            want = torch.where(seen.gather(-1, order), order, n).sort(-1).values
            want_s = torch.where(want < n, score.gather(-1, want.clamp(max=n - 1)), -math.inf)
            assert torch.equal(got[b, h], torch.where(want < n, want, -1).int())
            assert torch.equal(s[b, h], want_s)


@gpu
def test_select_by_parts_lists_what_each_token_alone_does():
    """Four parts of a chunk against calls of one query token each, whose
    scores do not depend on the split."""
    B, H, D, bt, top = 4, 8, 8, 16, 20
    T = 600_000  # 37500 blocks: 4.8 MB of scores a query token
    codes = torch.randint(-127, 128, (B, H, T // bt, 2, D), dtype=torch.int8, device="cuda",
                          generator=torch.Generator(device="cuda").manual_seed(4))
    scales = torch.rand((B, H, T // bt), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    q = queries(B, H, 700, D, torch.float16)  # 3.4 GB in one piece
    got, s = _lib.calls().block_select(codes, scales, bt, T, q, top, 1, 2, None, True)
    for i in (0, 1, 174, 175, 176, 349, 350, 524, 525, 699):  # the parts' ends, each token alone
        t = T - 700 + i + 1
        one, one_s = _lib.calls().block_select(codes, scales, bt, t, q[:, :, i:i + 1], top, 1, 2, None, True)
        assert torch.equal(got[:, :, i], one[:, :, 0]) and torch.equal(s[:, :, i], one_s[:, :, 0])


def test_c_alignment_refusals():
    """Vector accesses to pointers off their alignment would fault on the device: refused on the host."""
    L, d = _lib.lib(), ctypes.byref(_desc())
    for off in (1, 4, 8):
        assert L.cq_block_bounds(d, *{**BOUNDS, "codes": P + off}.values(), None) == -1
        assert L.cq_block_bounds_at(d, P, 1000, 1, 64, P + off, P, 16, None) == -1
        assert L.cq_block_bounds_read(P + off, P, 16, 16, 0, 4, 128, P, None) == -1
        assert L.cq_block_bounds_read(P, P, 16, 16, 0, 4, 128, P + off, None) == -1
        assert b"aligned" in L.cq_last_error()
    for off in (1, 2):
        assert L.cq_sparse_attention(d, *{**SPARSE_ARGS, "ws": P + off}.values(), None) == -1
        assert b"aligned" in L.cq_last_error()


@gpu
def test_offsets_past_32_bits():
    """A cache of 4.5 GB (four million tokens of 8 heads): its last tokens'
    ranges, lists and attention are those of a cache that holds them alone."""
    H, n, chunk, kw = 8, 62, 65536, dict(stride_k=64, stride_v=32, delta_bits_v=3)
    last = chunk + 333
    T, t0 = n * chunk + last, n * chunk
    big, tail = ChronoQuantCache(max_tokens=T, **kw), ChronoQuantCache(**kw)
    g = torch.Generator(device="cuda").manual_seed(7)
    k, v = (torch.randn((1, H, last, 128), generator=g, device="cuda").half() for _ in range(2))
    for i in range(n):
        big.update_and_fetch(k[:, :, :chunk] + i / 8, v[:, :, :chunk])
    big.update_and_fetch(k, v)
    tail.update_and_fetch(k, v)
    assert big.store.buf.numel() > 2 ** 32 and big.offset == T
    whole, part = BlockIndex(big, 64).update(), BlockIndex(tail, 64).update()
    assert torch.equal(whole.bounds(t0 // 64), part.bounds())
    whole.codes[:, :, t0 // 64:] = 0
    assert torch.equal(whole.update(t0).bounds(t0 // 64), part.bounds())
    for S in (1, 40):
        q = queries(1, 4 * H, S, 128, torch.bfloat16)
        got = whole.select(q, 12, starts=torch.tensor([t0], device="cuda"))
        want = part.select(q, 12)
        assert torch.equal(got, torch.where(want >= 0, want + t0 // 64, -1))
        assert torch.equal(chronoquant_sparse_sdpa(q, big, 0.1, got, 64), chronoquant_sparse_sdpa(q, tail, 0.1, want, 64))
