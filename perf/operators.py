"""Workloads of the sparse-attention path over a compressed KV cache: the plain form of each operator in elementary
torch operations, and the calls a program makes of this package's kernels.

Four operators (``op`` of a case):

``bounds``  per block of cached tokens and channel, the range of the decoded keys, held as int8 codes with one fp32
            scale per block: s = max|x| / 126, lower code floor(min x / s), upper code ceil(max x / s), x the fp16 keys
            fp16(anchor + fp16(code * scale)).  A case recomputes the blocks from token ``start`` on.
``select``  the blocks each query token attends to, per kv-head: query heads quantised to int8, the score of a block
            the largest over the group's heads of s_q * s_block * sum_d max(q_d * lo_d, q_d * hi_d) (whole numbers
            until the two scales), the first and the most recent visible blocks always taken, ties to the lowest index.
            The listed blocks' scores come with them (ranks that share a sequence merge their lists by these).
``sparse``  attention of each query token over the tokens of its listed blocks, keys and values decoded as
            anchor + code * scale; query * scale is rounded to the query's type, as everywhere in this package.
``rope``    RMSNorm of each query and key head, then the rotation of the first ``rot`` channels by position, from fused
            QKV rows to head-major queries and keys.
"""

import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda"


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # a 16384-token prompt of 8 sequences has just been encoded (Standard strides): all its blocks at once
        dict(name="bounds-prompt", op="bounds", B=8, H=8, T=16384, D=128, sk=32, sv=8, vbits=4, bt=64, start=0),
        # one long document (Full-Throttle strides) whose length is no multiple of anything, coarser blocks
        dict(name="bounds-long-odd", op="bounds", B=1, H=8, T=262139, D=128, sk=64, sv=32, vbits=3, bt=128, start=0),
        # a decode step: the block that the newest token fell into, of 16 sequences
        dict(name="bounds-step", op="bounds", B=16, H=8, T=32701, D=128, sk=64, sv=32, vbits=3, bt=64, start=32700),
        # one sequence, one new token: latency
        dict(name="select-step", op="select", B=1, H=8, G=4, S=1, T=8190, D=128, sk=32, sv=8, vbits=4, bt=64, top=32,
             first=1, recent=2, dtype="bf16", padded=False),
        # a serving batch with left padding at 32k tokens
        dict(name="select-batch", op="select", B=16, H=8, G=4, S=1, T=32768, D=128, sk=64, sv=32, vbits=3, bt=64,
             top=64, first=1, recent=2, dtype="bf16", padded=True),
        # one sequence of half a million tokens: 8192 blocks to choose from
        dict(name="select-long", op="select", B=1, H=8, G=4, S=1, T=524287, D=128, sk=64, sv=32, vbits=3, bt=64,
             top=128, first=1, recent=4, dtype="f16", padded=False),
        # a query chunk, each of its tokens with a list of its own
        dict(name="select-chunk", op="select", B=1, H=8, G=4, S=512, T=65536, D=128, sk=64, sv=32, vbits=3, bt=64,
             top=32, first=1, recent=2, dtype="bf16", padded=False),
        # the attention of the same three situations
        dict(name="sparse-step", op="sparse", B=1, H=8, G=4, S=1, T=8190, D=128, sk=32, sv=8, vbits=4, bt=64, top=32,
             dtype="bf16", padded=False),
        dict(name="sparse-batch", op="sparse", B=16, H=8, G=4, S=1, T=32768, D=128, sk=64, sv=32, vbits=3, bt=64,
             top=64, dtype="bf16", padded=True),
        dict(name="sparse-chunk", op="sparse", B=1, H=8, G=4, S=512, T=65536, D=128, sk=64, sv=32, vbits=3, bt=64,
             top=32, dtype="f16", padded=False),
        # a decode step's 32 rows at their own positions
        dict(name="rope-step", op="rope", B=32, S=1, H=8, G=4, D=128, rot=128, pairs="halves", dtype="bf16"),
        # a prompt of odd length behind a long context: angles of far positions
        dict(name="rope-prompt", op="rope", B=2, S=8191, H=8, G=4, D=128, rot=128, pairs="halves", dtype="bf16"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["bounds", "select", "select", "sparse", "sparse", "rope"])
    if op == "rope":
        D = rng.choice([64, 128, 128, 256])
        S = rng.choice([1, log(2, 8191)])
        H, G = rng.choice([2, 4, 8]), rng.choice([1, 2, 4, 7])
        most = 2 * 8191 * 40 * 128 // (H * (G + 1) * D)  # tokens of the largest listed case at this width
        S = min(S, most)
        B = min(log(1, 64) if S == 1 else log(1, 4), most // S)
        return dict(op=op, B=B, S=S, H=H, G=G, D=D, rot=rng.choice([D, D, D // 2]),
                    pairs=rng.choice(["halves", "halves", "adjacent"]), dtype=rng.choice(["bf16", "f16"]))
    sk, sv, vbits = rng.choice([(32, 8, 4), (64, 32, 3), (64, 32, 3), (16, 16, 4)])
    c = dict(op=op, D=128, sk=sk, sv=sv, vbits=vbits, bt=rng.choice([64, 64, 128, 256]), H=rng.choice([1, 2, 4, 8]))
    if op == "bounds":
        T = log(33, 220000)
        c.update(T=T, B=rng.randint(1, max(1, min(16, 8 * 8 * 16384 // (c["H"] * T)))),
                 start=rng.choice([0, 0, rng.randrange(T)]))
        return c
    S = rng.choice([1, 1, 1, log(2, 512)])
    T = S + log(1, 65000 if S > 1 else 260000)
    n = -(-T // c["bt"])
    first, recent = rng.choice([0, 1, 2]), rng.choice([1, 2, 3])
    top = max(first + recent, min(n + 1, log(3, 32 if S > 1 else 100)))
    top = min(top, max(first + recent, (32 if S > 1 else 64) * 64 // c["bt"]))
    cap = max(1, 16 * 8 * 32768 // (c["H"] * T))
    c.update(S=S, T=T, B=1 if S > 1 else rng.randint(1, min(16, cap)), G=rng.choice([1, 2, 4, 8]) if S == 1 else 4,
             top=top, dtype=rng.choice(["bf16", "f16"]), padded=S == 1 and rng.random() < 0.3)
    if op == "select":
        c.update(first=first, recent=recent)
    return c


# --------------------------------------------------------------------------- inputs
def _component(gen, B, H, T, D, stride, bits, spread):
    """One compressed component as a cache saves it: fp16 anchors with a few strong channels, packed residual codes
    and per-token scales, as the codec leaves them (codes within +-(2^(bits-1) - 1), the largest one used)."""
    nk = (T - 1) // stride + 1
    np_ = T - nk
    chan = torch.randn((1, H, 1, D), generator=gen, device=DEV) * spread
    kf = (chan + torch.randn((B, H, nk, D), generator=gen, device=DEV)).half()
    top = 2 ** (bits - 1) - 1
    packed = torch.empty((B, H, np_, D // 8), dtype=torch.int32, device=DEV)
    shift = torch.arange(0, 32, 4, device=DEV, dtype=torch.int32)
    for b in range(B):
        for h in range(H):
            c = (torch.randn((np_, D // 8, 8), generator=gen, device=DEV) * (top * 0.42)).round().clamp(-top, top)
            packed[b, h] = ((c.int() + 8) << shift).sum(-1, dtype=torch.int32)
    sc = (0.35 / top * torch.exp(0.3 * torch.randn((B, H, np_), generator=gen, device=DEV))).half()
    return kf, packed, sc


def _cache(gen, c):
    k = _component(gen, c["B"], c["H"], c["T"], c["D"], c["sk"], 4, 2.0)
    v = _component(gen, c["B"], c["H"], c["T"], c["D"], c["sv"], c["vbits"], 0.5)
    return k, v


def _starts(gen, c):
    """First real token of each sequence of a left-padded batch, or None."""
    if not c["padded"]:
        return None
    return torch.randint(0, max(1, c["T"] // 4), (c["B"],), generator=gen, device=DEV)


def _lists(gen, c, starts):
    """Block lists as a selection leaves them: ascending, the first and the newest visible blocks among them, the
    others drawn with a popularity that a head's queries share; -1 behind where fewer are visible."""
    B, H, S, T, bt, top = c["B"], c["H"], c["S"], c["T"], c["bt"], c["top"]
    n = -(-T // bt)
    j = torch.arange(n, device=DEV)
    last = (T - S + torch.arange(S, device=DEV)) // bt
    firstb = torch.zeros(B, dtype=torch.long, device=DEV) if starts is None else starts // bt
    w = torch.rand((B, H, 1, n), generator=gen, device=DEV) + 0.3 * torch.rand((B, H, S, n), generator=gen, device=DEV)
    w = torch.where((j == firstb[:, None])[:, None, None, :] | (j >= last[:, None] - 1)[None, None], w + 2.0, w)
    seen = (j <= last[:, None])[None, None] & (j >= firstb[:, None])[:, None, None, :]
    w = torch.where(seen, w, -1.0)
    k = min(top, n)
    val, idx = w.topk(k, -1)
    idx = torch.where(val >= 0, idx, n).sort(-1).values
    out = torch.full((B, H, S, top), -1, dtype=torch.int32, device=DEV)
    out[..., :k] = torch.where(idx < n, idx, -1).int()
    return out


def _queries(gen, c):
    Hq = c["H"] * c["G"]
    return (1.3 * torch.randn((c["B"], Hq, c["S"], c["D"]), generator=gen, device=DEV)).to(DT[c["dtype"]])


def _freqs(rot):
    return 1.0 / (1.0e6 ** (torch.arange(0, rot, 2, device=DEV, dtype=torch.float32) / rot))


def _rope_inputs(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    B, S, H, Hq, D, dt = c["B"], c["S"], c["H"], c["H"] * c["G"], c["D"], DT[c["dtype"]]
    qkv = torch.randn((B, S, (Hq + 2 * H) * D), generator=gen, device=DEV).to(dt)
    wq = (1 + 0.2 * torch.randn(D, generator=gen, device=DEV)).to(dt)
    wk = (1 + 0.2 * torch.randn(D, generator=gen, device=DEV)).to(dt)
    at = torch.randint(0, 500000, (B, 1), generator=gen, device=DEV)
    return dict(qkv=qkv, wq=wq, wk=wk, pos=at + torch.arange(S, device=DEV), inv_freq=_freqs(c["rot"]))


def _inputs(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = {}
    s["k"], s["v"] = _cache(gen, c)
    if c["op"] != "bounds":
        s["q"] = _queries(gen, c)
        s["starts"] = _starts(gen, c)
    if c["op"] == "sparse":
        s["blocks"] = _lists(gen, c, s["starts"])
    return s


def prepare(case, seed):
    c = case
    s = _rope_inputs(c, seed) if c["op"] == "rope" else _inputs(c, seed)
    s["case"] = c
    if own and c["op"] != "rope":  # the program's cache, restored from its saved state, and its index of blocks
        import chronoquant_mlx_b200 as cq
        cache = cq.ChronoQuantCache(stride_k=c["sk"], stride_v=c["sv"], delta_bits_v=c["vbits"])
        (kk, pk, ck), (kv, pv, cv) = s.pop("k"), s.pop("v")
        cache.state = [kk, kv, pk.view(torch.uint32), ck, pv.view(torch.uint32), cv]
        s["cache"] = cache
        if c["op"] in ("bounds", "select"):
            s["index"] = cq.BlockIndex(cache, c["bt"]).update()
    if not own and c["op"] == "select":  # the index a program keeps beside its cache
        s["codes"], s["scales"] = _plain_codes(s.pop("k"), c, 0)
        s.pop("v")
    return s


# --------------------------------------------------------------------------- plain forms
def _unpack(words):
    shift = torch.arange(0, 32, 4, device=words.device, dtype=torch.int32)
    return (((words.unsqueeze(-1) >> shift) & 15) - 8).flatten(-2)


def _plain_codes(k, c, start):
    """(codes [B, H, n, 2, D] as whole numbers in fp32, scales [B, H, n]) of the blocks from token ``start`` on."""
    kf, packed, sc = k
    B, H, T, D, sk, bt = c["B"], c["H"], c["T"], c["D"], c["sk"], c["bt"]
    t = torch.arange(start // bt * bt, T, device=DEV)
    a = t // sk
    pf = (t - a - 1).clamp(min=0)
    x = kf[:, :, a]
    if packed.shape[2]:
        r = _unpack(packed[:, :, pf]).half() * sc[:, :, pf].unsqueeze(-1)
        x = torch.where((t % sk == 0)[:, None], x, x + r)
    n = -(-t.numel() // bt)
    pad = n * bt - t.numel()
    lo = torch.nn.functional.pad(x, (0, 0, 0, pad), value=math.inf).view(B, H, n, bt, D).amin(3).float()
    hi = torch.nn.functional.pad(x, (0, 0, 0, pad), value=-math.inf).view(B, H, n, bt, D).amax(3).float()
    s = torch.maximum(lo.abs(), hi.abs()).amax(-1) / torch.full((), 126.0, device=DEV)
    d = torch.where(s > 0, s, 1.0).double().unsqueeze(-1)  # in 64 bits: quotients next to a whole number
    codes = torch.stack((torch.floor(lo.double() / d), torch.ceil(hi.double() / d)), 3).float()
    return codes, s


def _plain_bounds(s):
    c = s["case"]
    codes, scale = _plain_codes(s["k"], c, c["start"])
    return codes * scale[..., None, None]


def _plain_select(s):
    c, q = s["case"], s["q"].float()
    B, H, G, S, T, D, bt, top = c["B"], c["H"], c["G"], c["S"], c["T"], c["D"], c["bt"], c["top"]
    n = -(-T // bt)
    amax = q.abs().amax(-1, keepdim=True)
    q8 = torch.round(q * (torch.full((), 127.0, device=DEV) / amax)).view(B, H, G * S, D)
    sq = (amax / torch.full((), 127.0, device=DEV)).view(B, H, G * S, 1)
    lo, hi = s["codes"][..., 0, :], s["codes"][..., 1, :]
    dot = torch.matmul(q8.clamp(min=0), hi.transpose(-1, -2)) + torch.matmul(q8.clamp(max=0), lo.transpose(-1, -2))
    score = (sq * s["scales"].unsqueeze(2) * dot).view(B, H, G, S, n).amax(2)
    j = torch.arange(n, device=DEV)
    last = ((T - S + torch.arange(S, device=DEV)) // bt).view(1, 1, S, 1)
    firstb = 0 if s["starts"] is None else (s["starts"] // bt).view(B, 1, 1, 1)
    rank = torch.where((j < firstb + c["first"]) | (j > last - c["recent"]), math.inf, score)
    rank = torch.where((j <= last) & (j >= firstb), rank, -math.inf)
    val, idx = torch.sort(rank, dim=-1, descending=True, stable=True)
    k = min(top, n)
    idx = torch.where(val[..., :k] > -math.inf, idx[..., :k], n).sort(-1).values
    out = torch.full((B, H, S, top), -1, dtype=torch.int32, device=DEV)
    out[..., :k] = torch.where(idx < n, idx, -1).int()
    of = torch.gather(score, -1, out.long().clamp(min=0))
    return out, torch.where(out >= 0, of, -math.inf)


def _gather(comp, stride, t):
    """Decoded rows (fp32) of the tokens ``t`` [B, H, S, L] of a component."""
    kf, packed, sc = comp
    b = torch.arange(t.shape[0], device=DEV).view(-1, 1, 1, 1)
    h = torch.arange(t.shape[1], device=DEV).view(1, -1, 1, 1)
    a = t // stride
    x = kf[b, h, a].float()
    if packed.shape[2]:
        pf = (t - a - 1).clamp(min=0)
        r = _unpack(packed[b, h, pf]).float() * sc[b, h, pf].float().unsqueeze(-1)
        x = torch.where((t % stride == 0).unsqueeze(-1), x, x + r)
    return x


def _scaled(q, dt, scale):
    return (q * torch.full((), scale, dtype=dt, device=DEV)).float()  # rounded to the query's type, as the package does


def _plain_sparse(s):
    c, blocks = s["case"], s["blocks"]
    B, H, G, S, T, D = c["B"], c["H"], c["G"], c["S"], c["T"], c["D"]
    t = (blocks.long().unsqueeze(-1) * c["bt"] + torch.arange(c["bt"], device=DEV)).flatten(-2)
    at = (T - S + torch.arange(S, device=DEV)).view(1, 1, S, 1)
    ok = (t >= 0) & (t <= at)
    if s["starts"] is not None:
        ok &= t >= s["starts"].view(B, 1, 1, 1)
    t = t.clamp(0, T - 1)
    q = _scaled(s["q"], s["q"].dtype, D ** -0.5).view(B, H, G, S, D).transpose(2, 3)  # [B, H, S, G, D]
    w = torch.matmul(q, _gather(s["k"], c["sk"], t).transpose(-1, -2))
    w = torch.where(ok.unsqueeze(3), w, -math.inf)
    m = w.amax(-1, keepdim=True)
    p = torch.exp(w - torch.where(m > -math.inf, m, 0.0))
    o = torch.matmul(p, _gather(s["v"], c["sv"], t)) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.transpose(2, 3).reshape(B, H * G, S, D).to(s["q"].dtype)


def _rotate(x, cos, sin, c):
    """The first ``rot`` channels of x [B, S, heads, D] rotated, as halves or as adjacent pairs."""
    rot = c["rot"]
    r, rest = x[..., :rot], x[..., rot:]
    if c["pairs"] == "halves":
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((r, rest), -1)


def _plain_rope(s):
    c = s["case"]
    B, S, H, Hq, D = c["B"], c["S"], c["H"], c["H"] * c["G"], c["D"]
    x = s["qkv"].float().view(B, S, Hq + 2 * H, D)[:, :, :Hq + H]
    w = torch.cat((s["wq"].float().expand(Hq, D), s["wk"].float().expand(H, D)))
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
    ang = (s["pos"].double().unsqueeze(-1) * s["inv_freq"].double()).unsqueeze(2)  # in 64 bits: far positions
    y = _rotate(x, ang.cos().float(), ang.sin().float(), c).to(s["qkv"].dtype).transpose(1, 2)
    return y[:, :Hq].contiguous(), y[:, Hq:].contiguous()


def run(state):
    s, c = state, state["case"]
    if own:
        import chronoquant_mlx_b200 as cq
        if c["op"] == "bounds":
            return s["index"].update(c["start"]).bounds(c["start"] // c["bt"])
        if c["op"] == "select":
            return s["index"].select(s["q"], c["top"], first=c["first"], recent=c["recent"], starts=s["starts"],
                                     return_scores=True)
        if c["op"] == "sparse":
            return cq.chronoquant_sparse_sdpa(s["q"], s["cache"], c["D"] ** -0.5, s["blocks"], c["bt"],
                                              starts=s["starts"])
        return cq.qk_norm_rope(s["qkv"], c["H"] * c["G"], c["H"], s["inv_freq"], s["pos"], s["wq"], s["wk"], eps=1e-6,
                               pairs=c["pairs"])
    return {"bounds": _plain_bounds, "select": _plain_select, "sparse": _plain_sparse, "rope": _plain_rope}[c["op"]](s)


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "rope":
        n = c["B"] * c["S"] * c["H"] * (c["G"] + 1) * c["D"]
        return {"bytes": 4 * n + 8 * c["B"] * c["S"], "flops": 8 * n}
    units, D, T, bt = c["B"] * c["H"], c["D"], c["T"], c["bt"]

    def row(stride):  # bytes per token of one component
        return 2 * D / stride + (D / 2 + 2) * (1 - 1 / stride)

    if c["op"] == "bounds":
        t0 = c["start"] // bt * bt
        n = -(-(T - t0) // bt)
        return {"bytes": units * ((T - t0) * row(c["sk"]) + n * (2 * D + 4 + 8 * D)), "flops": 4 * units * (T - t0) * D}
    G, S = c["G"], c["S"]
    qo = c["B"] * c["H"] * G * S * D * 2
    if c["op"] == "select":
        n = -(-T // bt)
        return {"bytes": units * n * (2 * D + 4) + qo + units * S * c["top"] * 8, "flops": 2 * units * S * G * n * D}
    tokens = min(c["top"] * bt, T)
    return {"bytes": units * tokens * (row(c["sk"]) + row(c["sv"])) + 2 * qo + units * S * c["top"] * 4,
            "flops": 4 * units * S * G * tokens * D}


# --------------------------------------------------------------------------- the definitions in 64 bits
def _decoded(comp, b, h, stride, T, f):
    """Rows of one stream in 64 bits: ``f(anchor, code, scale)`` for residual tokens, the anchor for the others."""
    kf, packed, sc = (x[b, h] for x in comp)
    x = kf.double().repeat_interleave(stride, 0)[:T].clone()
    rest = torch.arange(T, device=DEV) % stride != 0
    code = torch.stack([(packed >> (4 * i)) & 15 for i in range(8)], -1).reshape(packed.shape[0], -1) - 8
    x[rest] = f(x[rest], code.double(), sc.double()[:, None])
    return x


def _exact_bounds(c, s, whole=False):
    """Ranges of the cache's fp16 keys; the scale a 32-bit number, the codes the nearest whole numbers outside (which
    come back themselves, with their scales, where ``whole``)."""
    b0, out = c["start"] // c["bt"], []

    def key(a, code, sc):
        return (a + (code * sc).half().double()).half().double()

    for b in range(c["B"]):
        for h in range(c["H"]):
            x = _decoded(s["k"], b, h, c["sk"], c["T"], key)
            part = [x[i:i + c["bt"]] for i in range(b0 * c["bt"], c["T"], c["bt"])]
            if len(part) > 1 and part[-1].shape[0] < c["bt"]:  # repeat a row: the range stays
                part[-1] = torch.cat((part[-1], part[-1][:1].expand(c["bt"] - part[-1].shape[0], -1)))
            part = torch.stack(part)
            lo, hi = part.amin(1), part.amax(1)
            unit = (torch.maximum(-lo, hi).amax(1) / 126).float()[:, None]
            codes = torch.stack((torch.floor(lo / unit.double()), torch.ceil(hi / unit.double())), 1)
            out.append((codes, unit[:, 0]) if whole else codes * unit.double()[:, None])
    if whole:
        return out
    return torch.stack(out).view(c["B"], c["H"], -1, 2, c["D"])


def _exact_select(c, s):
    """The listed blocks' scores in 64 bits; which blocks are listed goes by the 32-bit score of the definition."""
    B, H, G, S, T, top = c["B"], c["H"], c["G"], c["S"], c["T"], c["top"]
    n = -(-T // c["bt"])
    vals = _exact_bounds({**c, "start": 0}, s, whole=True)
    q = s["q"].float().view(B, H, G, S, -1)
    biggest = q.abs().amax(-1, keepdim=True)
    q8 = torch.round(q * torch.div(torch.tensor(127.0, device=DEV), biggest)).double()
    out = torch.full((B, H, S, top), -math.inf, dtype=torch.float64, device=DEV)
    for b in range(B):
        firstb = 0 if s["starts"] is None else int(s["starts"][b]) // c["bt"]
        for h in range(H):
            codes, unit = vals[b * H + h]
            per = [q8[b, h, g].clamp(min=0) @ codes[:, 1].T + q8[b, h, g].clamp(max=0) @ codes[:, 0].T
                   for g in range(G)]  # whole numbers
            sq = (biggest[b, h] / torch.tensor(127.0, device=DEV)).unbind(0)
            score = torch.stack([d * sq[g].double() * unit.double() for g, d in enumerate(per)]).amax(0)
            rank = torch.stack([(sq[g] * unit) * d.float() for g, d in enumerate(per)]).amax(0)
            last = (T - S + torch.arange(S, device=DEV)[:, None]) // c["bt"]
            j = torch.arange(n, device=DEV)[None]
            key = torch.where((j - firstb < c["first"]) | (last - j < c["recent"]), math.inf, rank)
            key[(j > last) | (j < firstb)] = -math.inf
            order = torch.argsort(-key, dim=1, stable=True)[:, :top]
            taken = torch.zeros_like(key, dtype=torch.bool).scatter_(1, order, True) & (key > -math.inf)
            for i in range(S):
                mine = score[i, taken[i]]  # in ascending order of the blocks
                out[b, h, i, :mine.numel()] = mine
    return None, out


def _exact_sparse(c, s):
    B, H, G, S, T, D = c["B"], c["H"], c["G"], c["S"], c["T"], c["D"]
    q = (s["q"] * torch.tensor(D ** -0.5, device=DEV).to(s["q"].dtype)).double().view(B, H, G, S, D)
    out = torch.zeros((B, H, G, S, D), dtype=torch.float64, device=DEV)
    within = torch.arange(c["bt"], device=DEV)
    for b in range(B):
        start = 0 if s["starts"] is None else s["starts"][b]
        for h in range(H):
            k = _decoded(s["k"], b, h, c["sk"], T, lambda a, code, sc: a + code * sc)
            v = _decoded(s["v"], b, h, c["sv"], T, lambda a, code, sc: a + code * sc)
            for i0 in range(0, S, 64):
                rows = torch.arange(i0, min(S, i0 + 64), device=DEV)
                t = (s["blocks"][b, h, rows].long()[:, :, None] * c["bt"] + within).flatten(1)
                ok = (t >= start) & (t >= 0) & (t <= (T - S + rows)[:, None])
                t = torch.where(ok, t, 0)
                w = torch.einsum("gsd,sld->gsl", q[b, h, :, rows], k[t])
                w = torch.where(ok, w, -math.inf)
                p = torch.nan_to_num(torch.softmax(w, -1), nan=0.0)
                out[b, h, :, rows] = torch.einsum("gsl,sld->gsd", p, v[t])
    return out.view(B, H * G, S, D)


def _exact_rope(c, s):
    B, S, H, Hq, D, rot = c["B"], c["S"], c["H"], c["H"] * c["G"], c["D"], c["rot"]
    x = s["qkv"].double().view(B, S, -1, D)
    ang = s["pos"].double()[..., None] * s["inv_freq"].double()
    z = torch.polar(torch.ones_like(ang), ang)
    got = []
    for lo, hi, w in ((0, Hq, s["wq"]), (Hq, Hq + H, s["wk"])):
        y = x[:, :, lo:hi]
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + 1e-6) * w.double()
        half = rot // 2
        re, im = (y[..., :half], y[..., half:rot]) if c["pairs"] == "halves" else (y[..., 0:rot:2], y[..., 1:rot:2])
        u = torch.complex(re.contiguous(), im.contiguous()) * z[:, :, None]
        y = y.clone()
        if c["pairs"] == "halves":
            y[..., :half], y[..., half:rot] = u.real, u.imag
        else:
            y[..., 0:rot:2], y[..., 1:rot:2] = u.real, u.imag
        got.append(y.transpose(1, 2))
    return tuple(got)


def exact(case, seed):
    c = case
    if c["op"] == "rope":
        return _exact_rope(c, _rope_inputs(c, seed))
    return {"bounds": _exact_bounds, "select": _exact_select, "sparse": _exact_sparse}[c["op"]](c, _inputs(c, seed))
