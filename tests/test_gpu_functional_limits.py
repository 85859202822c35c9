"""The teacher-forced operators at the limits of what their documentation allows: nothing to do, the largest sizes, values of the
type's lowest, rows that take part in nothing.  Bounds and references are those of test_gpu_functional.py."""
import math

import pytest
import torch

from test_gpu_functional_edges import poisoned  # noqa: F401
from test_gpu_functional import BF16, DEV, F, F32, U, attn_check, attn_inputs, attn_ref, attn_run, embed_inputs, gen, half, on, vocab_inputs, vocab_ref, vocab_run, within  # noqa: F401

pytestmark = pytest.mark.gpu


def nan(*shape, dtype=F32):
    return torch.full(shape, math.nan, dtype=dtype, device=DEV)


@pytest.mark.parametrize("V", [9, 1 << 18, (1 << 18) + 1, 1_000_003])
@pytest.mark.parametrize("positions", [0, 5])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_embedding_gradient_of_no_tokens_is_written(F, V, positions, dtype):  # noqa: F811
    """The entry point itself, on results full of NaN: no sequence of `positions` tokens, a vocabulary on both sides of the border of the
    two sorts."""
    import image_captioning_amd as m
    L, H = m._lib, 12
    code = L.F32 if dtype == F32 else L.BF16
    d, p = nan(V, H, dtype=dtype), nan(max(positions, 1), H, dtype=dtype)
    T = max(positions, 1)
    size = L.lib.mic_embed_grad_workspace_bytes(0, T, H, V, 1 if positions else 0)
    ws = torch.empty(max(size, 16), dtype=torch.uint8, device=DEV)
    L.check(L.lib.mic_embed_grad(None, 64, None, d.data_ptr(), p.data_ptr() if positions else None, code, code, 1.0, 0, T, H, V, ws.data_ptr(), size,
                                 torch.cuda.current_stream().cuda_stream), "mic_embed_grad")
    assert not d.isnan().any() and not d.any()
    assert not positions or (not p.isnan().any() and not p.any())
    none = torch.zeros(0, T, dtype=torch.long, device=DEV)
    for r in F.embedding_grad(torch.zeros(0, T, H, device=DEV, dtype=dtype), none, V, positions=positions):
        assert r is None or not r.any()


def test_embedding_with_the_most_words_there_can_be(F):  # noqa: F811
    """2^31 - 1 rows of one column: the last word and the first, and no token at all."""
    V = (1 << 31) - 1
    ids = torch.tensor([[V - 1, 0, 5, V - 1, 1 << 40]], device=DEV)
    g = torch.tensor([1.0, 2, 4, 8, 16], device=DEV).view(1, 5, 1).to(BF16)
    d, _ = F.embedding_grad(g, ids, V)
    assert int(torch.count_nonzero(d)) == 3
    assert [float(d[i, 0]) for i in (V - 1, 0, 5)] == [25.0, 2.0, 4.0]  # a word outside is the nearest one
    assert F.embedding_forward(ids, d).flatten().tolist() == [25.0, 2.0, 4.0, 25.0, 25.0]
    d.fill_(math.nan)
    del d
    d, _ = F.embedding_grad(g[:, :0], ids[:, :0], V)
    assert not torch.count_nonzero(d)


def test_vocab_loss_of_2_to_the_36_logits(F):  # noqa: F811
    """Narrow rows, so many of them that tiles of 64 x 64 would be 2^32 threads: some rows' results against their definition."""
    N, H, V = (1 << 24) + 3, 8, 4096
    g = torch.Generator(device=DEV).manual_seed(85)
    x = torch.randn(N, H, device=DEV, generator=g).to(BF16)
    w = torch.randn(V, H, device=DEV, generator=g).to(BF16)
    t = torch.randint(0, V, (N,), device=DEV, generator=g)
    loss, lse = F.vocab_loss_forward(x, w, t, ignore=(0,))
    rows = torch.cat([torch.tensor([0, 1, 63, 64, 127, 128, N - 4, N - 1]), torch.randint(0, N, (500,), generator=gen(86))])
    xs, ts = x[rows.to(DEV)].cpu(), t[rows.to(DEV)].cpu()
    a = torch.randn(N, device=DEV, generator=g)
    ref = vocab_ref(xs, w.cpu(), None, ts, a[rows.to(DEV)].cpu(), (0,), BF16)
    within(F.vocab_loss_grad(a, x, w, t, lse, ignore=(0,))[0][rows.to(DEV)], *ref["dx"], "dx")
    within(loss[rows.to(DEV)], *ref["loss"], "loss")
    within(lse[rows.to(DEV)], *ref["lse"], "lse")
    assert torch.isfinite(lse).all() and (lse > 0).all()


LOWEST = torch.finfo(F32).min


@pytest.mark.parametrize("N,H,V,dtype", [(256, 64, 24700, BF16), (2100, 136, 3119, BF16), (150, 96, 400, BF16), (150, 96, 400, F32)])
def test_vocab_loss_words_hidden_by_the_lowest_value(F, N, H, V, dtype):  # noqa: F811
    """A bias of the type's lowest value hides words like one of -infinity, also all words of a tile's columns; large and small tiles."""
    x, w, b, t, a = vocab_inputs(N, H, V, dtype, True, seed=80)
    hide = torch.rand(V, generator=gen(81)) < 0.2
    hide[64:330] = True
    hide[V - 70:] = True
    hide[:3] = False
    t = torch.where(hide[t], torch.full_like(t, 2), t)
    ref = vocab_ref(x, w, b.masked_fill(hide, -math.inf), t, a, (0,), dtype)
    got = vocab_run(F, *on(x, w, b.masked_fill(hide, LOWEST), t, a), (0,))
    for n in ("loss", "lse", "dx", "dw", "db"):
        within(got[n], *ref[n], n)
    same = vocab_run(F, *on(x, w, b.masked_fill(hide, -math.inf), t, a), (0,))
    for n in same:
        assert torch.equal(got[n], same[n]), n


BLIND = [
    # B, Tq, Tk, Hq, Hkv, D, how many of the first keys are hidden
    (2, 150, 100, 2, 1, 64, 0),     # more queries than keys: the first ones see nothing
    (2, 40, 30, 2, 2, 256, 0),      # the kernels for one tile of keys
    (3, 29, 29, 2, 2, 256, 11),     # captions padded on the left
    (3, 60, 60, 3, 1, 40, 33),
    (2, 300, 300, 2, 2, 128, 150),
    (2, 333, 333, 6, 2, 72, 47),    # three query heads to a key head
    (1, 520, 520, 2, 1, 32, 129),   # ranges of rows
    (1, 270, 270, 40, 1, 64, 5),    # more query heads than a tile of rows
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,Tq,Tk,Hq,Hkv,D,hidden", BLIND)
def test_attention_rows_that_see_nothing_may_hold_anything(F, B, Tq, Tk, Hq, Hkv, D, hidden, dtype):  # noqa: F811
    """Causal queries before the first key that is seen: what q and the output's gradient hold there enters no result."""
    q, k, v, go, _ = attn_inputs(B, Tq, Tk, Hq, Hkv, D, dtype, None, seed=82)
    m = None
    if hidden:
        m = (torch.arange(Tk) >= hidden).repeat(B, 1)
        if B > 1:
            m[-1] = True  # one sequence is not padded
        m[0, hidden + 1] = False
    first = [(int(m[b].int().argmax()) if hidden else 0) - (Tk - Tq) for b in range(B)]
    blind = torch.arange(Tq)[None] < torch.tensor(first)[:, None]
    assert blind.any() and not blind.all()
    ref = attn_ref(q, k, v, go, True, m, 1 / math.sqrt(D), dtype)
    bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).min])
    for seed, x in ((83, q), (84, go)):
        x[blind] = bad[torch.randint(0, 4, x[blind].shape, generator=gen(seed))].to(dtype)
    got = attn_run(F, *on(q, k, v, go), True, None if m is None else m.to(DEV))
    attn_check(got, ref)
    assert not got["o"][blind.to(DEV)].any() and not got["dq"][blind.to(DEV)].any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Tk", [20, 49, 130])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_sequence_without_a_key_may_hold_anything(F, Tk, causal, dtype):  # noqa: F811
    """All keys of one sequence are hidden: none of its inputs enters a result, and all its results are zero."""
    q, k, v, go, _ = attn_inputs(3, 40, Tk, 4, 2, 64, dtype, None, seed=87)
    m = torch.ones(3, Tk, dtype=torch.bool)
    m[1] = False
    ref = attn_ref(q, k, v, go, causal, m, 0.125, dtype)
    bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).min])
    for seed, x in ((88, q), (89, go), (90, k), (91, v)):
        x[1] = bad[torch.randint(0, 4, x[1].shape, generator=gen(seed))].to(dtype)
    got = attn_run(F, *on(q, k, v, go), causal, m.to(DEV))
    attn_check(got, ref)
    assert not any(got[n][1].any() for n in ("o", "dq", "dk", "dv"))


def test_attention_columns_past_32_bits_are_refused(F):  # noqa: F811
    q = torch.empty(0, 1, 1, 1 << 31, device=DEV)
    with pytest.raises(ValueError):
        F.attention_forward(q, q, q)
    with pytest.raises(ValueError):
        F.attention_grad(q, q, q, q, q, torch.empty(0, 1, 1, device=DEV))


@pytest.mark.parametrize("dtype,N,H,V", [(F32, 40_000, 72, 3500), (F32, 40_000, 41, 3500), (BF16, 90_000, 64, 3500), (F32, 1111, 300, 10007), (BF16, 2600, 520, 3500)])
@pytest.mark.parametrize("counted", [0.0, 0.01, 0.5, 1.0])
def test_vocab_loss_pieces_and_ranges(F, poisoned, dtype, N, H, V, counted):  # noqa: F811
    """Several pieces of the vocabulary, ranges of k in both products, and so many of the rows counted: partial sums share the scratch."""
    x, w, b, t, a = vocab_inputs(N, H, V, dtype, True, seed=90, ignore_share=0.0)
    t = torch.where(torch.rand(N, generator=gen(92)) < counted, t.clamp_min(1), torch.zeros_like(t))
    args = on(x, w, b, t, a / N)
    ref = {n: [v.cpu() for v in r] for n, r in vocab_ref(*args, (0,), dtype).items()}
    got = vocab_run(F, *args, (0,))
    for n, r in ref.items():
        within(got[n], *r, n)
    again = vocab_run(F, *args, (0,))
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_vocab_loss_one_gradient_for_every_row(F, dtype):  # noqa: F811
    """A scalar tensor, and the expanded one that a sum or a mean leaves: the bits that a gradient per row gives."""
    x, w, b, t, _ = vocab_inputs(70, 96, 500, dtype, True, seed=93)
    a = torch.full((70,), 0.37)
    ref = vocab_ref(x, w, b, t, a, (0,), dtype)
    args = on(x, w, b, t, a)
    rows = vocab_run(F, *args, (0,))
    for n, r in ref.items():
        within(rows[n], *r, n)
    scalar = vocab_run(F, *args[:4], torch.tensor(0.37, device=DEV), (0,))
    assert all(torch.equal(rows[n], scalar[n]) for n in rows)
    for scale, reduce in ((1.0, torch.sum), (70.0, torch.mean)):
        leaves = [v.clone().requires_grad_() for v in args[:3]]
        loss = reduce(F.vocab_loss(leaves[0], leaves[1], args[3], bias=leaves[2], ignore=(0,)))
        loss.backward(torch.tensor(scale, device=DEV))
        one = vocab_run(F, *args[:4], torch.tensor(1.0, device=DEV), (0,))
        for n, v in zip(("dx", "dw", "db"), leaves):
            if scale == 1.0:
                assert torch.equal(v.grad, one[n]), n
            else:  # 70 / 70 in fp32
                within(v.grad, *vocab_ref(x, w, b, t, torch.ones(70), (0,), dtype)[n], n)


def test_frozen_operands(F):  # noqa: F811
    """Gradients of what needs one, whichever that is, are those of the plain calls; what is frozen gets none."""
    ids, table, p, g = embed_inputs(3, 6, 11, 16, F32, F32, True, seed=94)
    ids, table, p, g = on(ids, table, p, g)
    d_table, d_pos = F.embedding_grad(g, ids, 11, scale=2.0, positions=6)
    for need in ((True, False), (False, True)):
        leaves = [v.clone().requires_grad_(n) for v, n in zip((table, p), need)]
        F.embedding(ids, *leaves, scale=2.0).backward(g)
        for v, n, r in zip(leaves, need, (d_table, d_pos)):
            assert torch.equal(v.grad, r) if n else v.grad is None
    q, k, v, go, _ = attn_inputs(2, 9, 70, 4, 2, 32, F32, None, seed=95)
    q, k, v, go = on(q, k, v, go)
    plain = attn_run(F, q, k, v, go, False, None)
    for need in ((True, False, False), (False, True, False), (False, False, True)):
        leaves = [x.clone().requires_grad_(n) for x, n in zip((q, k, v), need)]
        F.attention(*leaves).backward(go)
        for x, n, r in zip(leaves, need, ("dq", "dk", "dv")):
            assert torch.equal(x.grad, plain[r]) if n else x.grad is None
    x, w, b, t, a = on(*vocab_inputs(40, 32, 90, F32, True, seed=96))
    plain = vocab_run(F, x, w, b, t, a, (0,))
    for need in ((True, False, False), (False, True, False), (False, False, True)):
        leaves = [y.clone().requires_grad_(n) for y, n in zip((x, w, b), need)]
        F.vocab_loss(leaves[0], leaves[1], t, bias=leaves[2], ignore=(0,)).backward(a)
        for y, n, r in zip(leaves, need, ("dx", "dw", "db")):
            assert torch.equal(y.grad, plain[r]) if n else y.grad is None


# ---- tensors of more than 2^31 elements, and the longest of each size ------------------------------------------------------------
def test_attention_over_a_cache_past_32_bits(F):  # noqa: F811
    """One query on 2^24 + 5 keys of 128 columns: the last ones lie behind 2^31 elements.  A few keys, those among them, carry the softmax."""
    T, D = (1 << 24) + 5, 128
    scale, h = 1 / math.sqrt(D), 2.0 ** -9
    torch.manual_seed(100)
    q, g = (torch.randn(1, 1, 1, D, device=DEV).to(BF16) for _ in range(2))
    k, v = (torch.empty(1, T, 1, D, dtype=BF16, device=DEV).normal_(0, s) for s in (0.02, 1.0))
    heavy = torch.tensor([0, 1000, 1 << 23, (1 << 24) - 1, 1 << 24, T - 1], device=DEV)
    k[0, heavy, 0] += (torch.linspace(2.3, 2.6, 6, device=DEV)[:, None] * q[0, 0]).to(BF16)
    o, lse = F.attention_forward(q, k, v, causal=True)
    dq, dk, dv = F.attention_grad(g, q, k, v, o, lse, causal=True)
    Q, G = q.double().view(D), g.double().view(D)

    def blocks():
        for lo in range(0, T, 1 << 20):
            yield slice(lo, lo + (1 << 20)), k[0, lo:lo + (1 << 20), 0].double(), v[0, lo:lo + (1 << 20), 0].double()
    z = torch.cat([K @ Q for _, K, _ in blocks()]) * scale
    L = torch.logsumexp(z, 0)
    p = torch.exp(z - L)
    dP = torch.cat([V @ G for *_, V in blocks()])
    out, mag = sum(p[r] @ V for r, _, V in blocks()), sum(p[r] @ V.abs() for r, _, V in blocks())
    delta = (p * dP).sum()
    # a score is a sum of 128 products; a range's sum l takes at most 2^14 additions
    e = 2 * (D + 3) * U * scale * (k[0, heavy, 0].double().abs() @ Q.abs()).max() + 200 * U + 2.0 ** -10
    near = lambda got, ref, tol, what: within(got.reshape(ref.shape), ref.cpu(), 1.01 * tol.cpu() + 1e-30, what)  # noqa: E731
    near(lse, L.view(1), (e + 2 * U * L.abs()).view(1), "lse")
    near(o, out, (2 * h + 2 * e) * mag, "o")
    e_delta = (3 * h + 2 * e) * (mag @ G.abs())
    e_ds = p * ((h + e) * (dP - delta).abs() + e_delta + 200 * U * (dP.abs() + delta.abs()))
    ds = p * (dP - delta)
    near(dq, scale * sum(ds[r] @ K for r, K, _ in blocks()), scale * (1 + h) * sum((e_ds[r] + (h + e) * ds[r].abs()) @ K.abs() for r, K, _ in blocks()), "dq")
    rows = torch.cat([heavy, torch.randint(0, T, (1000,), device=DEV), torch.arange(T - 200, T, device=DEV)])
    near(dk[0, rows, 0], scale * ds[rows, None] * Q, scale * (e_ds + h * ds.abs())[rows, None] * (1 + h) * Q.abs(), "dk")
    near(dv[0, rows, 0], p[rows, None] * G, (2 * h + 2 * e) * p[rows, None] * G.abs(), "dv")
    light = torch.ones(T, dtype=torch.bool, device=DEV)
    light[heavy] = False
    assert float(dv[0, :, 0].abs().amax(1)[light].max()) <= 1.1 * float((p[light]).max() * G.abs().max())


def test_embedding_past_32_bits(F):  # noqa: F811
    """2^21 + 3 tokens of 1,024 columns: result and gradient have more than 2^31 elements."""
    n, H, V = (1 << 21) + 3, 1024, 1000
    torch.manual_seed(101)
    ids = torch.randint(0, V, (n,), device=DEV)
    table = torch.randn(V, H, device=DEV).to(BF16)
    out = F.embedding_forward(ids, table)
    assert all(torch.equal(out[lo:lo + (1 << 18)], table[ids[lo:lo + (1 << 18)]]) for lo in range(0, n, 1 << 18))
    d, _ = F.embedding_grad(out, ids, V, dtype=F32)  # the gradient of a word's row: its count times the row
    m = torch.bincount(ids, minlength=V).double()[:, None].cpu()
    ref = m * table.double().cpu()
    within(d, ref, 1.01 * ((m + 2) * U * ref.abs()) + 1e-30, "d_table")


def test_vocab_loss_rows_past_32_bits(F):  # noqa: F811
    """2^21 + 1 rows of 1,032 columns: x and dx have more than 2^31 elements."""
    N, H, V = (1 << 21) + 1, 1032, 260
    torch.manual_seed(102)
    x = torch.empty(N, H, dtype=BF16, device=DEV).normal_()
    w, b = (2 / math.sqrt(H) * torch.randn(V, H, device=DEV)).to(BF16), torch.randn(V, device=DEV)
    t = torch.randint(0, V, (N,), device=DEV)
    a = torch.randn(N, device=DEV) / N
    got = vocab_run(F, x, w, b, t, a, (0,))
    rows = torch.cat([torch.arange(130), torch.arange(N - 300, N), torch.randint(0, N, (300,), generator=gen(103))]).to(DEV)
    ref = vocab_ref(x[rows].cpu(), w.cpu(), b.cpu(), t[rows].cpu(), a[rows].cpu(), (0,), BF16)
    for n in ("loss", "lse", "dx"):
        within(got[n][rows], *ref[n], n)
    dw, db = torch.zeros(V, H, dtype=torch.float64, device=DEV), torch.zeros(V, dtype=torch.float64, device=DEV)
    mag_w, mag_b = torch.zeros_like(dw), torch.zeros_like(db)
    W, B = w.double().t().contiguous(), b.double()
    for lo in range(0, N, 1 << 17):
        r = slice(lo, lo + (1 << 17))
        X = x[r].double()
        d = torch.softmax(X @ W + B, 1)
        d[torch.arange(d.shape[0]), t[r]] -= 1
        d *= (a[r].double() * (t[r] != 0))[:, None]
        D = d.t().contiguous()
        dw += D @ X; db += d.sum(0)
        mag_w += D.abs() @ X.abs(); mag_b += d.abs().sum(0)
    # A logit: 1,035 U times sum |x w|, below 64 here.  A sum over the rows in fp32: at most 64 ranges of N / 64 / 64 tiles of 64 k, four additions each,
    # and the join; the column sums: 2^14 partial sums of 128 rows, by 16
    e = 2 * 1035 * U * 64 + 400 * U
    within(got["dw"], dw.cpu(), (1.01 * ((half(BF16) + e + 2200 * U) * mag_w + half(BF16) * dw.abs())).cpu(), "dw")
    within(got["db"], db.cpu(), (1.01 * (e + 1300 * U) * mag_b).cpu(), "db")


@pytest.mark.parametrize("N,H,V,dtype", [(3, 8, (1 << 23) + 5, BF16), (5, (1 << 20) + 8, 7, BF16), (70, (1 << 18) + 4, 40, F32), ((1 << 20) + 9, 12, 33, F32)])
def test_vocab_loss_with_one_very_long_size(F, N, H, V, dtype):  # noqa: F811
    g = torch.Generator(device=DEV).manual_seed(104)
    x = torch.randn(N, H, device=DEV, generator=g).to(dtype)
    w = (2.0 / math.sqrt(H) * torch.randn(V, H, device=DEV, generator=g)).to(dtype)
    t, a = torch.randint(0, V, (N,), device=DEV, generator=g), torch.randn(N, device=DEV, generator=g)
    got = vocab_run(F, x, w, None, t, a, ())
    ref = vocab_ref(x, w, None, t, a, (), dtype)
    for n, r in ref.items():
        if r is not None:
            within(got[n], r[0].cpu(), r[1].cpu(), n)


@pytest.mark.parametrize("dtype,N,H,V", [(BF16, 2600, 520, 3500), (F32, 700, 96, 4000)])
def test_vocab_loss_in_a_graph_with_other_rows_counted(F, dtype, N, H, V):  # noqa: F811
    """How many rows count is known on the device alone: one capture, replayed for none, one, some and all of them."""
    x, w, b, t, a = on(*vocab_inputs(N, H, V, dtype, True, seed=97, ignore_share=0.0))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        vocab_run(F, x, w, b, t, a, (0,))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = vocab_run(F, x, w, b, t, a, (0,))
    words = t.clamp_min(1)
    for seed, share in enumerate((0.5, 0.0, 1.0, 1.5 / N, 0.1)):
        rows = torch.rand(N, generator=gen(98 + seed)) < share
        t.copy_(torch.where(rows.to(DEV), words, torch.zeros_like(words)))
        graph.replay()
        eager = vocab_run(F, x, w, b, t, a, (0,))
        torch.cuda.synchronize()
        assert all(torch.equal(held[n], eager[n]) for n in held), share


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_left_padding_in_a_graph(F, dtype):  # noqa: F811
    """One capture, replayed for other paddings: rows without a key hold NaN."""
    q, k, v, go, _ = on(*attn_inputs(2, 90, 90, 4, 2, 64, dtype, None, seed=99))
    m = torch.ones(2, 90, dtype=torch.bool, device=DEV)
    Q, G = q.clone(), go.clone()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        attn_run(F, Q, k, v, G, True, m)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = attn_run(F, Q, k, v, G, True, m)
    for hidden in ((0, 0), (3, 61), (89, 1), (33, 90)):
        m.copy_(torch.arange(90, device=DEV)[None] >= torch.tensor(hidden, device=DEV)[:, None])
        for x, y in ((Q, q), (G, go)):
            x.copy_(y.masked_fill(~m[:, :, None, None], math.nan))
        graph.replay()
        torch.cuda.synchronize()
        attn_check(held, attn_ref(q.cpu(), k.cpu(), v.cpu(), go.cpu(), True, m.cpu(), 0.125, dtype))
