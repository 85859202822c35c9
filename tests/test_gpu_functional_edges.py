"""The teacher-forced operators where they can go wrong: borders of tiles, chunks and plans, poisoned scratch memory, odd addresses,
values that must not matter.  Bounds and references are those of test_gpu_functional.py."""
import math

import pytest
import torch

from test_gpu_functional import (BF16, DEV, F, F32, U, attn_check, attn_inputs, attn_ref, attn_run, embed_grad_ref, embed_inputs, gen,  # noqa: F401
                                 half, on, vocab_check, vocab_inputs, vocab_ref, vocab_run, within)

pytestmark = pytest.mark.gpu


@pytest.fixture
def poisoned(F, monkeypatch):  # noqa: F811
    """Scratch memory of exactly the size asked for, full of NaN, with a border behind it that nobody may touch."""
    held = []

    def workspace(size, like):
        if size == 0:
            return None, 0
        t = torch.full((size + 4096,), 0xFF, dtype=torch.uint8, device=like.device)
        held.append((t, size))
        return t, t.data_ptr()
    monkeypatch.setattr(F, "_workspace", workspace)
    yield held
    torch.cuda.synchronize()
    assert held and all((t[size:] == 0xFF).all() for t, size in held)


def embed_check(F, ids, g, V, scale, odt, T):  # noqa: F811
    d, dp = F.embedding_grad(g.to(DEV), ids.to(DEV), V, scale=scale, positions=T, dtype=odt)
    ref, mag, m = embed_grad_ref(ids.long(), g, V, scale)
    within(d, ref, 1.01 * ((m + 2) * U * mag + half(odt) * ref.abs()) + 1e-30, "table")
    g64 = g.double()
    within(dp, g64.sum(0), 1.01 * (g.shape[0] * U * g64.abs().sum(0) + half(odt) * g64.sum(0).abs()) + 1e-30, "pos")


@pytest.mark.parametrize("n", [1, 15, 16, 17, 63, 64, 65, 8191, 8192, 8193])
def test_embedding_around_the_borders(F, poisoned, n):  # noqa: F811
    """One word for every token and two alternating ones; token counts around a chunk, a wave and the border of the two sorts."""
    g = torch.randn(1, n, 24, generator=gen(n)).to(BF16)
    embed_check(F, torch.full((1, n), 3, dtype=torch.int32), g, 9, 2.0, F32, n)
    embed_check(F, (torch.arange(n) % 2 * 8)[None], g, 9, -0.5, BF16, n)


@pytest.mark.parametrize("B,T,V,H", [(3, 50, 70, 40), (5, 2000, 300000, 16), (700, 30, 3500, 72)])
def test_embedding_in_poisoned_scratch(F, poisoned, B, T, V, H):  # noqa: F811
    ids, _, _, g = embed_inputs(B, T, V, H, F32, BF16, True, seed=40, hot=0.4)
    embed_check(F, ids, g, V, 1.0, F32, T)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H", [64, 33])
def test_embedding_off_a_16_byte_boundary(F, dtype, H):  # noqa: F811
    """Table, positions and the output's gradient begin one element behind a 16-byte boundary."""
    ids, table, pos, g = embed_inputs(4, 21, 50, H, dtype, dtype, True, seed=41)

    def off(t):
        flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device=DEV)
        flat[1:] = t.to(DEV).reshape(-1)
        return flat[1:].view(t.shape)
    got = F.embedding_forward(ids.int().to(DEV), off(table), off(pos), scale=0.5, dtype=F32)
    assert torch.equal(got.cpu(), 0.5 * table.float()[ids] + pos.float())
    aligned = F.embedding_grad(g.to(DEV), ids.to(DEV), 50, positions=21, dtype=F32)
    for a, b in zip(aligned, F.embedding_grad(off(g), ids.to(DEV), 50, positions=21, dtype=F32)):
        assert torch.equal(a, b)


def test_sizes_past_32_bits_are_refused(F):  # noqa: F811
    many = 1 << 32
    row = torch.zeros(1, 8, device=DEV)
    ids = torch.zeros(1, 2, dtype=torch.long, device=DEV)
    with pytest.raises(ValueError):
        F.embedding_forward(ids, row.expand(many, 8))
    with pytest.raises(ValueError):
        F.embedding_grad(torch.zeros(1, 2, 8, device=DEV), ids, many)
    x = torch.zeros(1, 1, 1, 8, device=DEV)
    with pytest.raises(ValueError):
        F.attention_forward(x, x.expand(1, many, 1, 8), x.expand(1, many, 1, 8))
    with pytest.raises(ValueError):
        F.vocab_loss_forward(row, row.expand(many, 8), ids[0, :1])


EDGES = [
    # B, Tq, Tk, Hq, Hkv, D, causal, mask
    (1, 40, 90, 6, 2, 64, True, "holes"),       # three query heads to a key head: tiles begin inside a position
    (1, 3, 80, 1100, 1, 32, False, "padded"),   # more query heads than one tile of rows
    (2, 2, 50, 40, 1, 40, True, None),
    (1, 150, 100, 2, 1, 256, True, "holes"),    # the first queries see no key
    (1, 5, 600, 2, 1, 256, True, None),         # few rows: ranges of keys in both directions
    (1, 1, 2500, 1, 1, 8, True, "holes"),
    (1, 520, 520, 2, 1, 128, True, None),       # ranges of rows, more of them for the first keys
    (1, 900, 129, 1, 1, 64, True, "padded"),
    (2, 127, 128, 1, 1, 24, True, None),
    (1, 128, 64, 4, 4, 128, True, "holes"),
    (3, 31, 32, 2, 1, 16, True, "padded"),
    (300, 33, 20, 1, 1, 32, False, "padded"),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,Tq,Tk,Hq,Hkv,D,causal,mask", EDGES)
def test_attention_edges(F, poisoned, B, Tq, Tk, Hq, Hkv, D, causal, mask, dtype):  # noqa: F811
    poisoned.append((torch.full((1,), 0xFF, dtype=torch.uint8, device=DEV), 0))  # (small forwards need none)
    q, k, v, go, m = attn_inputs(B, Tq, Tk, Hq, Hkv, D, dtype, mask, seed=50)
    ref = attn_ref(q, k, v, go, causal, m, 1 / math.sqrt(D), dtype)
    attn_check(attn_run(F, *on(q, k, v, go), causal, None if m is None else m.to(DEV)), ref)


def test_attention_one_key_many_times(F):  # noqa: F811
    """The same key at every position, and the same heads for every query head: equal probabilities, gradients that add up."""
    q, k, v, go, _ = attn_inputs(2, 70, 140, 4, 1, 64, F32, None, seed=51)
    k, v = k[:, :1].expand(2, 140, 1, 64), v[:, :1].expand(2, 140, 1, 64)
    ref = attn_ref(q, k, v, go, False, None, 0.125, F32)
    D = [t.to(DEV) for t in (q, k[:, :1], v[:, :1], go)]
    attn_check(attn_run(F, D[0], D[1].expand(2, 140, 1, 64), D[2].expand(2, 140, 1, 64), D[3], False, None), ref)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N", [20, 64, 65, 300])
def test_vocab_loss_rows_that_do_not_count_may_hold_anything(F, poisoned, N, dtype):  # noqa: F811
    x, w, b, t, a = vocab_inputs(N, 96, 200, dtype, True, seed=60)
    ref = vocab_ref(x, w, b, t, a, (0,), dtype)
    hidden = t == 0
    assert hidden.any() and not hidden.all()
    bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).min])
    fill = bad[torch.randint(0, 4, x.shape, generator=gen(61))].to(dtype)
    a = torch.where(hidden, torch.full_like(a, math.nan), a)
    got = vocab_run(F, *on(torch.where(hidden[:, None], fill, x), w, b, t, a), (0,))
    count = ~hidden
    within(got["lse"][count.to(DEV)], ref["lse"][0][count], ref["lse"][1][count], "lse")
    for n in ("loss", "dx", "dw", "db"):
        within(got[n], *ref[n], n)


@pytest.mark.parametrize("N,H,V,bias,dtype", [(1, 64, 300, True, BF16), (70, 40, 1000, True, F32), (513, 72, 1031, False, BF16), (1111, 100, 2000, True, F32),
                                             (4200, 64, 2100, True, BF16)])
def test_vocab_loss_in_poisoned_scratch(F, poisoned, N, H, V, bias, dtype):  # noqa: F811
    x, w, b, t, a = vocab_inputs(N, H, V, dtype, bias, seed=62)
    vocab_check(vocab_run(F, *on(x, w, b, t.int(), a), (0,)), vocab_ref(x, w, b, t, a, (0,), dtype))


@pytest.mark.parametrize("counted", [0, 1, 257, 4000])
def test_vocab_loss_counted_rows_of_many(F, poisoned, counted):  # noqa: F811
    """The large tiles: so many of 4,200 rows count."""
    x, w, b, _, a = vocab_inputs(4200, 64, 2100, BF16, True, seed=63)
    t = torch.zeros(4200, dtype=torch.long)
    t[torch.randperm(4200, generator=gen(64))[:counted]] = torch.randint(1, 2100, (counted,), generator=gen(65))
    got = vocab_run(F, *on(x, w, b, t, a), (0,))
    vocab_check(got, vocab_ref(x, w, b, t, a, (0,), BF16))
    assert not got["dx"][(t == 0).to(DEV)].any()


def test_vocab_loss_one_row_many_times(F):  # noqa: F811
    """The same row, word and target everywhere."""
    x, w, b, t, a = vocab_inputs(400, 64, 300, F32, True, seed=66)
    x, t = x[:1].expand(400, 64), torch.full_like(t, 7)
    got = vocab_run(F, x[:1].to(DEV).expand(400, 64), *on(w, b, t, a), ())
    vocab_check(got, vocab_ref(x, w, b, t, a, (), F32))


def test_gradients_of_the_differentiable_calls_in_a_graph(F):  # noqa: F811
    """torch.autograd.grad through all three, captured and replayed with other inputs while nothing eager of the same leaves is alive."""
    def step(ids, table, w, t):
        h = F.embedding(ids, table).view(2, 40, 2, 32)
        o = F.attention(h, h, h, causal=True)
        loss = F.vocab_loss(o.reshape(80, 64), w, t, ignore=(0,)).sum()
        return (loss.detach(), *torch.autograd.grad(loss, (table, w)))

    def inputs(seed):
        g = gen(seed)
        return (torch.randint(0, 90, (2, 40), generator=g).to(DEV), torch.randn(90, 64, generator=g).to(BF16).to(DEV),
                torch.randn(90, 64, generator=g).to(BF16).to(DEV), torch.randint(0, 90, (80,), generator=g).to(DEV))
    held = inputs(70)
    leaves = [held[0], held[1].requires_grad_(), held[2].requires_grad_(), held[3]]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step(*leaves)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*leaves)
    for seed in (71, 72, 73):
        other = inputs(seed)
        with torch.no_grad():
            for a, b in zip(leaves, other):
                a.copy_(b)
        graph.replay()
        eager = step(other[0], other[1].requires_grad_(), other[2].requires_grad_(), other[3])
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b)


@pytest.mark.parametrize("N,H,V,bias", [(130, 100, 50021, True), (2100, 136, 3119, False), (257, 70, 26001, True), (60, 96, 9001, True), (127, 64, 52000, False)])
def test_vocab_loss_around_the_large_tiles(F, poisoned, N, H, V, bias):  # noqa: F811
    """bf16 on both sides of the rule for the large tiles, edges of every kind."""
    x, w, b, t, a = vocab_inputs(N, H, V, BF16, bias, seed=67)
    vocab_check(vocab_run(F, *on(x, w, b, t, a), (0,)), vocab_ref(x, w, b, t, a, (0,), BF16))


def test_embedding_positions_of_a_very_long_sequence(F):  # noqa: F811
    """More columns to sum over sequences than one launch has workgroups for: each takes several.  One sequence: the sum is the gradient."""
    T, H = 1 << 17, 1032
    g = torch.randn(1, T, H, device=DEV, dtype=BF16)
    ids = torch.randint(0, 5, (1, T), device=DEV)
    _, dp = F.embedding_grad(g, ids, 5, positions=T)
    assert torch.equal(dp, g[0])
