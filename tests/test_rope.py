"""qk_norm_rope against 64 bits.

Bar: half a step of the output type, plus the fp32 arithmetic: the mean of D
squares (at most D/2 + 1 roundings of 2^-24 on its root), the reciprocal root,
two products, the angle's reduction (pi * 2^-24), sine and cosine (2 steps) and
the rotation, in all at most (D/2 + 20) * 2^-24 of |a| + |b| of the pair."""

import math
from fractions import Fraction

import pytest
import torch

from chronoquant_mlx_b200 import _lib, qk_norm_rope

gpu = pytest.mark.gpu


def reference(qkv, Hq, Hkv, inv_freq, pos, wq, wk, eps, pairs):
    B, S, width = qkv.shape
    D = width // (Hq + 2 * Hkv)
    half = inv_freq.shape[0]
    ang = pos.double().expand(B, S)[..., None] * inv_freq.double()
    cos, sin = ang.cos()[:, :, None], ang.sin()[:, :, None]
    out, mag = [], []
    for a, b, w in ((0, Hq, wq), (Hq, Hq + Hkv, wk)):
        x = qkv.double()[..., a * D:b * D].reshape(B, S, b - a, D)
        if w is not None:
            x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w.double()
        y, m = x.clone(), x.abs().clone()
        lo, hi = ((slice(0, half), slice(half, 2 * half)) if pairs == "halves" else
                  (slice(0, 2 * half, 2), slice(1, 2 * half, 2)))
        y[..., lo] = x[..., lo] * cos - x[..., hi] * sin
        y[..., hi] = x[..., hi] * cos + x[..., lo] * sin
        m[..., lo] = m[..., hi] = x[..., lo].abs() + x[..., hi].abs()
        out.append(y.transpose(1, 2))
        mag.append(m.transpose(1, 2))
    return out, mag


def inputs(B, S, Hq, Hkv, D, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = (1.7 * torch.randn((B, S, (Hq + 2 * Hkv) * D), generator=g, device="cuda")).to(dtype)
    w = [(1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dtype) for _ in range(2)]
    return qkv, w[0], w[1]


def freqs(rot, theta=1e6):
    return 1.0 / (theta ** (torch.arange(0, rot, 2, device="cuda", dtype=torch.float32) / max(rot, 1)))


def check(got, ref, mag, D):
    half = torch.finfo(got[0].dtype).eps / 2
    for x, y, m in zip(got, ref, mag):
        assert x.shape == y.shape and x.is_contiguous()
        fp32 = (D / 2 + 20) * 2.0 ** -24 * m
        tol = half * (y.abs() + fp32) + fp32 + 2.0 ** -25  # fp16 results below 2^-14 step by 2^-24
        assert ((x.double() - y).abs() <= tol).all(), float(((x.double() - y).abs() / tol).max())


@gpu
@pytest.mark.parametrize("pairs", ["halves", "adjacent"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [  # B, S, Hq, Hkv, D, rot
    (1, 1, 1, 1, 128, 128), (3, 5, 8, 2, 128, 128), (2, 33, 7, 1, 64, 64), (1, 9, 4, 4, 256, 256), (2, 3, 5, 5, 72, 72),
    (1, 17, 6, 2, 128, 64), (2, 2, 3, 1, 96, 24), (1, 4, 2, 1, 8, 8), (1, 3, 4, 2, 128, 0), (32, 1, 32, 8, 128, 128)])
def test_matches_64_bits(shape, dtype, pairs):
    B, S, Hq, Hkv, D, rot = shape
    qkv, wq, wk = inputs(B, S, Hq, Hkv, D, dtype, seed=S)
    pos = torch.randint(0, 600000, (B, S), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    f = freqs(rot)
    check(qk_norm_rope(qkv, Hq, Hkv, f, pos, wq, wk, eps=1e-6, pairs=pairs),
          *reference(qkv, Hq, Hkv, f, pos, wq, wk, 1e-6, pairs), D)
    check(qk_norm_rope(qkv, Hq, Hkv, f, pos, pairs=pairs), *reference(qkv, Hq, Hkv, f, pos, None, None, 0, pairs), D)


@gpu
def test_positions_broadcast_far_and_negative():
    """One position for all, one per sequence, one per token, positions past
    2^31 and negative ones; a position of zero rotates nothing."""
    qkv, wq, wk = inputs(2, 4, 4, 2, 128, torch.float32)
    f = freqs(128)
    for pos in (torch.tensor(12345, device="cuda"), torch.tensor([[7], [3 * 10 ** 9]], device="cuda"),
                torch.tensor([1, 0, -5, 2 ** 40], device="cuda"), torch.arange(8, device="cuda").view(2, 4)):
        p = pos.expand(2, 4)
        check(qk_norm_rope(qkv, 4, 2, f, pos, wq, wk), *reference(qkv, 4, 2, f, p, wq, wk, 1e-6, "halves"), 128)
    plain = qk_norm_rope(qkv, 4, 2, f, torch.zeros(1, 1, dtype=torch.int64, device="cuda"))
    assert torch.equal(plain[0], qkv[..., :512].view(2, 4, 4, 128).transpose(1, 2))


@gpu
def test_strided_rows_and_odd_values():
    """Rows cut out of a wider buffer and off 16-byte alignment, channels that
    are not contiguous, an all-zero head (stays zero), inputs left as they were."""
    qkv, wq, wk = inputs(2, 3, 4, 2, 128, torch.bfloat16)
    qkv[0, 0, :128] = 0
    f, pos = freqs(128), torch.arange(3, device="cuda")
    want = qk_norm_rope(qkv, 4, 2, f, pos, wq, wk)
    assert not want[0][0, 0, 0].any()
    wide = torch.full((2, 5, 1024 + 67), 9.0, dtype=torch.bfloat16, device="cuda")
    cut = wide[:, 1:4, 65:65 + 1024]
    cut.copy_(qkv)
    before = wide.clone()
    odd = torch.empty(2 * 3 * 2048, dtype=torch.bfloat16, device="cuda").view(2, 3, 2048)[..., ::2]
    odd.copy_(qkv)
    off = [torch.empty(129, dtype=torch.bfloat16, device="cuda")[1:].copy_(w) for w in (wq, wk)]
    for x in (cut, odd):
        for a, b in zip(qk_norm_rope(x, 4, 2, f, pos, *off), want):
            assert torch.equal(a, b)
    assert torch.equal(wide, before)


@gpu
def test_empty_and_captured():
    f = freqs(128)
    q, k = qk_norm_rope(torch.empty((0, 4, 1024), device="cuda"), 4, 2, f, torch.arange(4, device="cuda"))
    assert q.shape == (0, 4, 4, 128) and k.shape == (0, 2, 4, 128)
    q, k = qk_norm_rope(torch.empty((2, 0, 1024), device="cuda"), 4, 2, f, torch.zeros((2, 0), dtype=torch.int64,
                                                                                         device="cuda"))
    assert q.shape == (2, 4, 0, 128)
    qkv, wq, wk = inputs(2, 3, 4, 2, 128, torch.bfloat16)
    pos = torch.zeros((2, 3), dtype=torch.int64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = qk_norm_rope(qkv, 4, 2, f, pos, wq, wk)
    pos.copy_(torch.tensor([[4, 5, 6], [100, 101, 102]]))
    graph.replay()
    for a, b in zip(out, qk_norm_rope(qkv, 4, 2, f, pos, wq, wk)):
        assert torch.equal(a, b)


@gpu
def test_refusals():
    qkv, wq, wk = inputs(2, 3, 4, 2, 128, torch.bfloat16)
    f, pos = freqs(128), torch.arange(3, device="cuda")
    good = dict(qkv=qkv, n_q_heads=4, n_kv_heads=2, inv_freq=f, positions=pos, q_weight=wq, k_weight=wk)
    for over in (dict(qkv=qkv[0]), dict(n_q_heads=5), dict(n_kv_heads=0), dict(inv_freq=f.double()),
                 dict(inv_freq=f.cpu()), dict(inv_freq=freqs(258)), dict(positions=pos.int()),
                 dict(positions=pos.cpu()), dict(q_weight=None), dict(q_weight=wq[:64]), dict(k_weight=wk.float()),
                 dict(k_weight=wk.cpu()), dict(pairs="other")):
        with pytest.raises(ValueError):
            qk_norm_rope(**{**good, **over})
    with pytest.raises(RuntimeError):
        qk_norm_rope(**{**good, "positions": torch.arange(4, device="cuda")})
    with pytest.raises(TypeError):
        qk_norm_rope(**{**good, "qkv": qkv.double()})
    with pytest.raises(NotImplementedError):
        qk_norm_rope(torch.zeros((1, 1, 3 * 12), device="cuda"), 1, 1, freqs(4), pos[:1])


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA"):
        qk_norm_rope(torch.zeros((1, 1, 384)), 1, 1, torch.zeros(64), torch.zeros((1, 1), dtype=torch.int64))


P = 0x10000
ARGS = dict(qkv=P, sb=1024, ss=1024, B=1, S=1, Hq=4, Hkv=2, D=128, rot=128, adj=0, wq=P, wk=P, f=P, pos=P, psb=0, pss=0,
            eps=1e-6, q=P, k=P, dt=1)


@pytest.mark.parametrize("over,status", [
    (dict(qkv=None), -1), (dict(q=None), -1), (dict(k=None), -1), (dict(wq=None), -1), (dict(wk=None), -1),
    (dict(f=None), -1), (dict(pos=None), -1), (dict(B=-1), -1), (dict(S=-1), -1), (dict(Hq=0), -1), (dict(Hkv=0), -1),
    (dict(D=12), -2), (dict(D=264), -2), (dict(rot=130), -1), (dict(rot=3), -1), (dict(rot=-2), -1), (dict(dt=3), -2)])
def test_c_refusals(over, status):
    assert _lib.lib().cq_qk_norm_rope_rows(*{**ARGS, **over}.values(), None) == status


def test_c_nothing_to_do():
    assert _lib.lib().cq_qk_norm_rope_rows(*{**ARGS, "B": 0}.values(), None) == 0


def test_c_too_many_heads():
    for over in (dict(Hq=2 ** 31 - 1), dict(Hkv=2 ** 30)):
        assert _lib.lib().cq_qk_norm_rope_rows(*{**ARGS, **over}.values(), None) == -2


PI = Fraction(314159265358979323846264338327950288419716939937510582097494459230781640628620899, 10 ** 80)


@gpu
@pytest.mark.parametrize("pairs", ["halves", "adjacent"])
@pytest.mark.parametrize("D", [128, 72])
def test_angles_of_positions_up_to_2_to_53(pairs, D):
    """Positions whose product with a frequency has more bits than a double:
    the angles are exact fractions here, reduced by 80 digits of pi."""
    pos = [2 ** 30 + 7, 2 ** 40 + 12345, -(2 ** 45) - 3, 2 ** 50 - 77, 2 ** 53 - 1, -(2 ** 53)]
    qkv = inputs(1, len(pos), 4, 2, D, torch.float32)[0]
    f = freqs(D)
    turns = [[Fraction(p) * Fraction(x) / (2 * PI) for x in f.tolist()] for p in pos]
    ang = torch.tensor([[float((t - round(t)) * 2 * PI) for t in row] for row in turns], device="cuda",
                       dtype=torch.float64)
    cos, sin = ang.cos()[None, :, None], ang.sin()[None, :, None]
    ref, mag = [], []
    for a, b in ((0, 4), (4, 6)):
        x = qkv.double()[..., a * D:b * D].reshape(1, len(pos), b - a, D)
        lo, hi = ((slice(0, D // 2), slice(D // 2, D)) if pairs == "halves" else (slice(0, D, 2), slice(1, D, 2)))
        y, m = torch.empty_like(x), torch.empty_like(x)
        y[..., lo] = x[..., lo] * cos - x[..., hi] * sin
        y[..., hi] = x[..., hi] * cos + x[..., lo] * sin
        m[..., lo] = m[..., hi] = x[..., lo].abs() + x[..., hi].abs()
        ref.append(y.transpose(1, 2))
        mag.append(m.transpose(1, 2))
    check(qk_norm_rope(qkv, 4, 2, f, torch.tensor(pos, device="cuda"), pairs=pairs), ref, mag, D)


@gpu
@pytest.mark.parametrize("Hkv", [8, 7])
def test_offsets_past_32_bits(Hkv):
    """Rows past 2^32 bytes (and 2^31 elements) of a prompt: the last ones come out as they do alone."""
    S, Hq, D = 400_000, 32, 128
    width = (Hq + 2 * Hkv) * D
    qkv = torch.empty((1, S, width), dtype=torch.bfloat16, device="cuda")
    assert qkv.numel() > 2 ** 31
    qkv[:, -50:] = inputs(1, 50, Hq, Hkv, D, torch.bfloat16)[0]
    qkv[:, :-50] = 1
    _, wq, wk = inputs(1, 1, 1, 1, D, torch.bfloat16)
    f, pos = freqs(D), torch.arange(S, device="cuda")
    got = qk_norm_rope(qkv, Hq, Hkv, f, pos, wq, wk)
    want = qk_norm_rope(qkv[:, -50:], Hq, Hkv, f, pos[-50:], wq, wk)
    for a, b in zip(got, want):
        assert torch.equal(a[:, :, -50:], b)
