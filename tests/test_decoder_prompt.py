"""The decoder's prompt path and its block-sparse steps.

Bars as in test_decoder.py: the same kernels in another order within 1e-3
relative (L2) of each other; the prompt path against one-token steps within
2e-2 (bf16 activations, other GEMM shapes, the query-chunk attention's fp16
reconstruction against the decode kernel's fp32 one)."""

import math

import pytest
import torch

from chronoquant_mlx_b200 import BlockIndex, chronoquant_sparse_sdpa, decoder
from chronoquant_mlx_b200.decoder import DecoderConfig, Qwen3StyleDecoder
from test_sparse import check_attention, decoded, ref_bounds, ref_select, ref_sparse

gpu = pytest.mark.gpu

CFG = DecoderConfig(layers=2, hidden=512, heads=8, kv_heads=2, head_dim=128, ffn=1024, vocab=1000)
FT = dict(stride_k=64, stride_v=32, delta_bits_v=3, dead_zone_v=0.05)


def rel(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


def prompt(B, S, seed=0):
    return torch.randint(0, CFG.vocab, (B, S), generator=torch.Generator().manual_seed(seed))


@gpu
@pytest.mark.parametrize("kw", [dict(), FT])
def test_prefill_matches_steps(kw):
    """A 70-token prompt in one chunk, in chunks of 33, and its last 3 tokens as
    single steps (eager and captured): the same logits, greedy ids and caches."""
    ids = prompt(2, 70)
    a, b, c = (Qwen3StyleDecoder(CFG, 2, 120, kw, seed=3) for _ in range(3))
    la = a.prefill(ids)
    lb = b.prefill(ids, chunk=33)
    assert rel(lb, la) < 2e-2
    c.prefill(ids[:, :67])
    for t in range(67, 69):
        c.ids.copy_(ids[:, t])
        c.step_eager()
        for L in c.layers:  # eager steps advance the device length; the host's follows
            L["cache"].offset += 1
    c.capture()
    c.ids.copy_(ids[:, 69])
    lc = c.decode(1)
    assert rel(lc, la) < 2e-2
    assert a.layers[1]["cache"].offset == b.layers[1]["cache"].offset == c.layers[1]["cache"].offset == 70
    assert int(a.pos) == int(c.pos) == 70 and int(a.layers[0]["len"][0]) == int(c.layers[0]["len"][0]) == 70
    assert torch.equal(a.ids, la.argmax(-1))
    # the first layer's K/V depend on the ids and positions alone, up to the rounding of two norm kernels
    for x, y in zip(a.layers[0]["cache"].reconstruct_history(), c.layers[0]["cache"].reconstruct_history()):
        assert rel(x, y) < 1e-2
    c.prefill(prompt(2, 2))
    with pytest.raises(RuntimeError):  # the captured step held the lengths of before
        c.decode(1)
    more = prompt(2, 5, seed=1)  # a second prompt behind the first
    assert rel(a.prefill(more), Qwen3StyleDecoder(CFG, 2, 120, kw, seed=3).prefill(torch.cat((ids, more), 1))) < 2e-2


@gpu
@pytest.mark.parametrize("kw", [dict(), FT, dict(stride_k=12, stride_v=4)])
def test_sparse_step_over_every_block_is_the_dense_step(kw):
    """With room for every block the sparse decoder is the dense one: eager
    steps for every layout, captured ones too, across a block's end."""
    T0 = 317
    dense_ok = kw.get("stride_k") != 12  # the dense step needs the decode kernel's layouts
    d = Qwen3StyleDecoder(CFG, 2, T0 + 10, kw, seed=3)
    s = Qwen3StyleDecoder(CFG, 2, T0 + 10, kw, seed=3, sparse=dict(top=6))
    for m in (d, s):
        m.fill_context(T0)
    if not dense_ok:
        d._attention = None
    s.capture() if dense_ok else None
    for i in range(6):
        ids = torch.tensor([5 + i, 77 - i], device="cuda")
        s.ids.copy_(ids)
        d.ids.copy_(ids)
        ls = (s.decode(1) if dense_ok else s.step_eager()).float().clone()
        if dense_ok:
            assert rel(ls, d.step_eager()) < 1e-2
        assert torch.isfinite(ls).all()
        n = T0 + i + 1
        want = list(range(-(-n // 64))) + [-1] * (6 - -(-n // 64))
        assert s.blocks[0, 0, 0].tolist() == want
    assert int(s.layers[1]["len"][0]) == T0 + 6


@gpu
def test_sparse_steps_follow_their_index():
    """Captured sparse steps with few blocks: every layer attends to what a
    fresh index over its cache selects (the eager path's own calls), and
    graph and eager agree."""
    T0, kw, sp = 900, FT, dict(top=5, block_tokens=64, first=1, recent=1)
    g = Qwen3StyleDecoder(CFG, 2, T0 + 80, kw, seed=7, sparse=sp)
    e = Qwen3StyleDecoder(CFG, 2, T0 + 80, kw, seed=7)
    for m in (g, e):
        m.fill_context(T0)
    g.capture()

    def attend(L, q, k, v):
        cache = L["cache"]
        cache.update_and_fetch(k.unsqueeze(2), v.unsqueeze(2))
        blocks = BlockIndex(cache, 64).select(q.unsqueeze(2), 5, first=1, recent=1)
        L["blocks"] = blocks
        return chronoquant_sparse_sdpa(q.unsqueeze(2), cache, 1 / math.sqrt(128), blocks, 64).squeeze(2)

    for i in range(70):  # past a block's end
        ids = torch.tensor([i, 3 * i], device="cuda")
        g.ids.copy_(ids)
        e.ids.copy_(ids)
        lg, le = g.decode(1).float().clone(), e.step_eager(attend).float()
        assert rel(lg, le) <= 1e-3, i
        assert torch.equal(g.blocks, e.layers[-1]["blocks"]), i  # the last layer's lists
    for L in g.layers:
        whole = BlockIndex(L["cache"], 64).update()
        n = whole.n_blocks
        assert L["index"].covered == T0 + 70 and torch.equal(L["index"].codes[:, :, :n], whole.codes[:, :, :n])
    # an eager call on the same index afterwards goes on from there
    assert g.layers[0]["index"].select(torch.zeros((2, 8, 1, 128), device="cuda").bfloat16(), 5).shape == (2, 2, 1, 5)


@gpu
def test_sparse_prefill():
    """A long prompt through the sparse path: its first chunk is dense, the
    later ones select; the result is close to the dense model's, the lists hold
    their own block."""
    ids = prompt(1, 600, seed=2)
    dense = Qwen3StyleDecoder(CFG, 1, 700, FT, seed=3).prefill(ids, chunk=200)
    m = Qwen3StyleDecoder(CFG, 1, 700, FT, seed=3, sparse=dict(top=8, block_tokens=64))
    got = m.prefill(ids, chunk=200)
    assert torch.isfinite(got).all() and rel(got, dense) < 0.5  # 8 of 10 blocks: another, nearby function
    all_blocks = Qwen3StyleDecoder(CFG, 1, 700, FT, seed=3, sparse=dict(top=8, block_tokens=96 * 2))
    assert rel(all_blocks.prefill(ids, chunk=200), dense) < 2e-2


def test_refusals():
    for sparse in (dict(), dict(first=1), dict(top=4, blocks=3), dict(top=4, recent=0)):
        with pytest.raises(ValueError):
            Qwen3StyleDecoder(CFG, 1, 64, sparse=sparse, device="cpu")
    with pytest.raises(NotImplementedError):
        Qwen3StyleDecoder(CFG, 1, 64, sparse=dict(top=4), seq_group=object(), device="cpu")


@gpu
def test_prefill_refusals():
    m = Qwen3StyleDecoder(CFG, 2, 64, seed=3)
    for ids in (prompt(1, 4), prompt(2, 4)[:, :0], prompt(2, 4)[0], prompt(2, 65)):
        with pytest.raises(ValueError):
            m.prefill(ids)
    with pytest.raises(RuntimeError):
        m.decode(1)
    m.seq_group = object()
    with pytest.raises(NotImplementedError):
        m.prefill(prompt(2, 4))


@gpu
def test_a_new_context_drops_the_captured_step():
    """A captured step holds the lengths and buffers of the context it was
    captured over: a context filled in afterwards needs another capture."""
    for sparse in (None, dict(top=4)):
        m = Qwen3StyleDecoder(CFG, 2, 200, FT, seed=3, sparse=sparse)
        m.fill_context(100)
        m.capture()
        m.fill_context(20)
        with pytest.raises(RuntimeError, match="capture"):
            m.decode(1)
        m.capture()
        assert torch.isfinite(m.decode(2)).all()
        assert m.layers[1]["cache"].offset == int(m.layers[1]["len"][0]) == 122


@gpu
@pytest.mark.parametrize("sparse", [None, dict(top=6)])
def test_prompts_and_eager_steps_in_turn(sparse):
    """Eager steps advance the length on the device alone; a prompt behind them
    goes on from there, and so does a filled-in context."""
    ids = prompt(2, 75)
    whole = Qwen3StyleDecoder(CFG, 2, 120, FT, seed=3).prefill(ids)
    m = Qwen3StyleDecoder(CFG, 2, 120, FT, seed=3, sparse=sparse)
    m.prefill(ids[:, :60])
    for t in range(60, 63):
        m.ids.copy_(ids[:, t])
        m.step_eager()
    m.prefill(ids[:, 63:70])
    assert m.layers[0]["cache"].offset == m.layers[1]["cache"].offset == int(m.pos) == 70
    m.ids.copy_(ids[:, 70])
    m.step_eager()
    got = m.prefill(ids[:, 71:])
    assert rel(got, whole) < 2e-2
    for L in m.layers:
        assert L["cache"].offset == int(L["len"][0]) == 75
        assert sparse is None or L["index"].covered == 75
    # a caller's own attention appends through the cache: its offset is the length then
    def attend(L, q, k, v):
        L["cache"].update_and_fetch(k.unsqueeze(2), v.unsqueeze(2))
        return q
    m.step_eager(attend)
    m.prefill(ids[:, :2])
    assert m.layers[1]["cache"].offset == int(m.layers[1]["len"][0]) == int(m.pos) == 78
    # another state restored into the caches is what the next prompt follows, however short
    for L in m.layers:
        c = type(L["cache"])(**FT)
        c.update_and_fetch(*(torch.randn((2, 2, 40, 128), device="cuda").bfloat16() for _ in range(2)))
        L["cache"].state = c.state
    m.prefill(ids[:, :2])
    assert m.layers[1]["cache"].offset == int(m.layers[1]["len"][0]) == int(m.pos) == 42
    m.step_eager()
    m.fill_context(5)
    assert m.layers[1]["cache"].offset == int(m.layers[1]["len"][0]) == 48


@gpu
@pytest.mark.parametrize("sparse", [None, dict(top=4, block_tokens=32)])
def test_a_prompt_that_failed_can_be_run_again(sparse, monkeypatch):
    """An error inside a chunk (no memory, say) leaves every layer's cache and
    index at the length before the prompt."""
    ids = prompt(2, 90)
    a, b = (Qwen3StyleDecoder(CFG, 2, 200, FT, seed=3, sparse=sparse) for _ in range(2))
    for m in (a, b):
        m.fill_context(150 - 40)
    attend, seen = b._chunk_attention, []

    def fail(L, q):
        seen.append(q.shape[2])
        out = attend(L, q)
        if len(seen) == 4:  # the second layer of the second chunk
            raise torch.cuda.OutOfMemoryError("no memory")
        return out

    monkeypatch.setattr(b, "_chunk_attention", fail)
    with pytest.raises(torch.cuda.OutOfMemoryError):
        b.prefill(ids, chunk=40)
    for L in b.layers:
        assert L["cache"].offset == 110
        if sparse:
            fresh = BlockIndex(L["cache"], 32).update()
            assert torch.equal(L["index"].update().bounds(), fresh.bounds()) and L["index"].covered == 110
    assert torch.equal(b.prefill(ids, chunk=30), a.prefill(ids, chunk=30))
    for x, y in zip(a.layers, b.layers):
        assert x["cache"].offset == y["cache"].offset == 200
        for s, t in zip(x["cache"].state, y["cache"].state):
            assert torch.equal(s.view(torch.uint8), t.view(torch.uint8))
        assert sparse is None or torch.equal(x["index"].bounds(), y["index"].bounds())


@gpu
@pytest.mark.parametrize("cfg,kw", [(CFG, dict(stride_k=12, stride_v=4)),
                                    (DecoderConfig(layers=2, hidden=512, heads=32, kv_heads=2, head_dim=128, ffn=1024,
                                                   vocab=1000), FT)])
def test_sparse_steps_of_other_layouts_are_captured(cfg, kw):
    """Layouts and groups (of 16 heads) that the dense decode kernel does not
    take: a sparse step needs none of it, captured steps are the eager ones."""
    T0, sp = 300, dict(top=4, block_tokens=32)
    g, e = (Qwen3StyleDecoder(cfg, 2, T0 + 40, kw, seed=3, sparse=sp) for _ in range(2))
    for m in (g, e):
        m.fill_context(T0)
    g.capture()
    for i in range(30):  # past a block's end
        ids = torch.tensor([5 + i, 77 - i], device="cuda")
        g.ids.copy_(ids)
        e.ids.copy_(ids)
        lg, le = g.decode(1).float().clone(), e.step_eager().float()
        assert rel(lg, le) <= 1e-3, i
        assert torch.equal(g.blocks, e.blocks), i
    assert g.layers[1]["cache"].offset == int(g.layers[1]["len"][0]) == T0 + 30


def test_prefill_refuses_ids_outside_the_vocabulary():
    """An embedding row that is not there would end the process's GPU context: refused on the host."""
    m = Qwen3StyleDecoder(CFG, 2, 64, device="cpu")
    good = prompt(2, 4)
    for bad in (-1, -CFG.vocab, CFG.vocab, 2 ** 40):
        ids = good.clone()
        ids[1, 2] = bad
        with pytest.raises(ValueError, match="outside"):
            m.prefill(ids)
    for dtype in (torch.float32, torch.bool, torch.uint8):  # masks, to an indexing
        with pytest.raises(TypeError, match="int32 or int64"):
            m.prefill((good > 0).to(dtype))
    assert m.layers[0]["cache"].offset == 0


@gpu
@pytest.mark.parametrize("kw,cfg", [(FT, CFG), (dict(), CFG), (dict(stride_k=12, stride_v=4), CFG),
                                    (FT, DecoderConfig(layers=2, hidden=512, heads=18, kv_heads=2, head_dim=128,
                                                       ffn=1024, vocab=1000))])
def test_sparse_prompt_chunks_against_64_bits(kw, cfg, monkeypatch):
    """Every chunk of a prompt, layer by layer: dense attention while the lists
    hold every block, then the lists of the definition over the layer's own cache
    and 64-bit attention over them, each row's own block among them."""
    sp = dict(top=5, block_tokens=64, first=1, recent=2)
    m = Qwen3StyleDecoder(cfg, 2, 700, kw, seed=3, sparse=sp)
    attend, select_blocks, seen = m._chunk_attention, [], []
    sparse_sdpa = decoder.chronoquant_sparse_sdpa

    def listed(q, cache, scale, blocks, bt, **rest):
        select_blocks.append(blocks)
        return sparse_sdpa(q, cache, scale, blocks, bt, **rest)

    def checked(L, q):
        before = len(select_blocks)
        out = attend(L, q)
        cache = L["cache"]
        T, S = cache.offset, q.shape[2]
        if T <= 5 * 64:
            assert len(select_blocks) == before
        else:
            assert len(select_blocks) == before + 1
            blocks = select_blocks[-1]
            codes, scales = ref_bounds(decoded(cache, fp16_keys=True)[0], 64)
            assert torch.equal(blocks.cpu(), ref_select(codes, scales, q, T, 64, 5, 1, 2)[0])
            own = (T - S + torch.arange(S, device="cuda")) // 64
            assert (blocks == own[:, None]).any(-1).all()
            ref, _, vmax = ref_sparse(*decoded(cache), q, 128 ** -0.5, blocks, 64)
            check_attention(out, ref, vmax)
        seen.append((T, len(select_blocks) - before))
        return out

    monkeypatch.setattr(decoder, "chronoquant_sparse_sdpa", listed)
    monkeypatch.setattr(m, "_chunk_attention", checked)
    got = m.prefill(prompt(2, 333, seed=5), chunk=111)
    assert torch.isfinite(got).all()
    got = m.prefill(prompt(2, 217, seed=6), chunk=120)
    assert torch.isfinite(got).all()
    assert seen == [(t, int(t > 320)) for t in (111, 222, 333, 453, 550) for _ in range(2)]


@gpu
@pytest.mark.parametrize("kw", [FT, dict(stride_k=12, stride_v=4)])
def test_sparse_prompt_over_every_block_is_the_dense_prompt(kw, monkeypatch):
    """Chunks sent through selection and sparse attention with room for every
    block: 64-bit attention over the whole cache, layer by layer, each over its own
    cache.  The first layer's keys and values are the dense decoder's bit for bit;
    the next layer's are not comparable in the end (a rounding of the first one's
    output moves codes next to a border by a whole step, a third of the largest
    residual in 3 bits)."""
    m = Qwen3StyleDecoder(CFG, 2, 500, kw, seed=3, sparse=dict(top=8, block_tokens=64))
    ran = []

    def sparse(L, q):
        cache, index = L["cache"], m._index(L)
        blocks = index.select(q, 8)
        S, T = q.shape[2], cache.offset
        own = (T - S + torch.arange(S, device="cuda")) // 64
        j = torch.arange(8, device="cuda")
        assert torch.equal(blocks[1, 1], torch.where(j <= own[:, None], j, -1).int())
        out = chronoquant_sparse_sdpa(q, cache, 128 ** -0.5, blocks, 64)
        ref, _, vmax = ref_sparse(*decoded(cache), q, 128 ** -0.5, blocks, 64)
        check_attention(out, ref, vmax)
        ran.append(T)
        return out

    monkeypatch.setattr(m, "_chunk_attention", sparse)
    ids = prompt(2, 450, seed=5)
    dense = Qwen3StyleDecoder(CFG, 2, 500, kw, seed=3)
    assert torch.isfinite(m.prefill(ids, chunk=150)).all() and torch.isfinite(dense.prefill(ids, chunk=150)).all()
    for x, y in zip(m.layers[0]["cache"].state, dense.layers[0]["cache"].state):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert ran == [150, 150, 300, 300, 450, 450]


def test_sparse_options_that_no_step_could_take_are_refused():
    """At once, not by the first prompt that grows past its lists."""
    for sparse in (dict(top=2), dict(top=4, first=2, recent=3), dict(top=0), dict(top=-3), dict(top=5000),
                   dict(top=8, first=-1), dict(top=8, block_tokens=0), dict(top=8, block_tokens=40),
                   dict(top=8, block_tokens=-16)):
        with pytest.raises(ValueError):
            Qwen3StyleDecoder(CFG, 1, 64, sparse=sparse, device="cpu")
    m = Qwen3StyleDecoder(CFG, 1, 64, sparse=dict(top=3, block_tokens=16), device="cpu")
    assert m.sparse == dict(top=3, block_tokens=16, first=1, recent=2)


@gpu
@pytest.mark.parametrize("sparse", [None, dict(top=4)])
def test_steps_over_moved_storage_are_refused(sparse):
    """Steps hold addresses of the caches' pages (a captured one of the indexes
    too): a restored state, pages that had to grow or an index that moved."""
    def fresh():
        m = Qwen3StyleDecoder(CFG, 2, 300, FT, seed=3, sparse=sparse)
        m.fill_context(100)
        m.capture()
        m.decode(1)
        return m

    m = fresh()
    other = type(m.layers[1]["cache"])(**FT)
    other.update_and_fetch(*(torch.randn((2, 2, 40, 128), device="cuda").bfloat16() for _ in range(2)))
    m.layers[1]["cache"].state = other.state
    for step in (lambda: m.decode(1), m.step_eager, m.capture):
        with pytest.raises(RuntimeError, match="moved"):
            step()
    m = fresh()
    m.layers[0]["cache"].update_and_fetch(*(torch.randn((2, 2, 700, 128), device="cuda").bfloat16() for _ in range(2)))
    for step in (lambda: m.decode(1), m.step_eager, m.capture):
        with pytest.raises(RuntimeError, match="moved"):
            step()
    m = fresh()
    before = m.layers[1]["cache"].offset
    if sparse:
        m.layers[1]["index"].reserve(5000)
        with pytest.raises(RuntimeError, match="moved"):
            m.decode(1)
        assert m.layers[1]["cache"].offset == before
        m.capture()
    assert torch.isfinite(m.decode(3)).all()


@gpu
def test_a_context_filled_in_behind_another_goes_on_from_its_position():
    """The next step's position is the number of tokens cached, however they came there."""
    m = Qwen3StyleDecoder(CFG, 2, 200, FT, seed=3)
    m.fill_context(60)
    assert int(m.pos) == 60
    m.step_eager()
    m.fill_context(30)
    assert int(m.pos) == m.layers[0]["cache"].offset == int(m.layers[0]["len"][0]) == 91


@gpu
def test_prefill_refuses_layers_of_different_lengths():
    """A state restored into some layers only: no position fits them all."""
    m = Qwen3StyleDecoder(CFG, 2, 200, FT, seed=3)
    m.prefill(prompt(2, 50))
    other = type(m.layers[1]["cache"])(**FT)
    other.update_and_fetch(*(torch.randn((2, 2, 40, 128), device="cuda").bfloat16() for _ in range(2)))
    m.layers[1]["cache"].state = other.state
    for call in (lambda: m.prefill(prompt(2, 5)), lambda: m.fill_context(5)):
        with pytest.raises(RuntimeError, match="different lengths"):
            call()
    m.layers[0]["cache"].state = other.state
    m.prefill(prompt(2, 5))
    assert m.layers[0]["cache"].offset == m.layers[1]["cache"].offset == 45
