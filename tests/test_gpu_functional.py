"""The teacher-forced operators against their definitions in 64 bits on the CPU.

Tolerances are bounds, not fits: u = 2^-24 is half a step of fp32, h = finfo(dtype).eps / 2 half a step of the result's type.  A
sum of m terms in fp32, in any order, is off by at most m * u * (sum of the terms' magnitudes), up to terms of order u^2."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def F():
    import image_captioning_amd as m
    return m.functional


def half(dtype):
    return torch.finfo(dtype).eps / 2


def within(got, ref, tol, what=""):
    """|got - ref| <= tol elementwise; got may be on the GPU, ref and tol are fp64 on the CPU."""
    got = got.double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((got - ref).abs().max()), float((((got - ref).abs()) / tol.clamp_min(1e-300)).max()))


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- embedding ----------------------------------------------------------------------------------------------------------
def embed_inputs(B, T, V, H, tdt, odt, pos, seed=0, hot=None):
    g = gen(seed)
    ids = torch.randint(0, V, (B, T), generator=g)
    if hot is not None:  # one word takes most of the tokens
        ids = torch.where(torch.rand(B, T, generator=g) < hot, torch.full_like(ids, V // 2), ids)
    return (ids, torch.randn(V, H, generator=g).to(tdt), torch.randn(T, H, generator=g).to(tdt) if pos else None,
            torch.randn(B, T, H, generator=g).to(odt))


def embed_grad_ref(ids, g, V, scale):
    H = g.shape[-1]
    flat, gd = ids.reshape(-1), g.double().reshape(-1, H)
    ref = torch.zeros(V, H, dtype=torch.float64).index_add_(0, flat, gd) * scale
    mag = torch.zeros(V, H, dtype=torch.float64).index_add_(0, flat, gd.abs()) * abs(scale)
    m = torch.bincount(flat, minlength=V).double()[:, None]
    return ref, mag, m


EMBED = [
    # B, T, V, H, table, out, positions, scale, share of one hot word
    (1, 1, 300, 64, F32, F32, False, 1.0, None),
    (3, 1, 1, 8, F32, BF16, True, 0.5, None),            # one word only
    (768, 1, 3500, 512, F32, BF16, False, 1.0, None),
    (64, 30, 3500, 512, F32, BF16, True, 1.0, 0.6),
    (7, 61, 1009, 300, F32, F32, True, 1.7320508, 0.3),   # H not a multiple of eight
    (5, 77, 513, 33, BF16, BF16, True, 3.0, 0.2),
    (2, 1500, 70000, 136, BF16, BF16, False, 11.5, 0.4),  # two sort passes, nearly every row empty
    (2, 4099, 300, 1032, BF16, F32, False, 32.0, 0.1),
    (40, 517, 262145, 16, F32, F32, False, 1.0, 0.05),    # three passes of the sort
    (1030, 2, 40, 72, BF16, BF16, True, 1.0, 0.9),        # sum over many sequences: the sliced column sum
]


@pytest.mark.parametrize("B,T,V,H,tdt,odt,pos,scale,hot", EMBED)
def test_embedding(F, B, T, V, H, tdt, odt, pos, scale, hot):
    ids, table, p, g = embed_inputs(B, T, V, H, tdt, odt, pos, hot=hot)
    scale = float(torch.tensor(scale, dtype=F32))
    ref = table.double()[ids] * scale
    mag = ref.abs()
    if pos:
        ref, mag = ref + p.double(), mag + p.double().abs()
    out = F.embedding_forward(ids.to(DEV), table.to(DEV), None if p is None else p.to(DEV), scale=scale, dtype=odt)
    assert out.dtype == odt
    within(out, ref, 1.01 * (2 * U * mag + half(odt) * ref.abs()), "out")
    for dt, width in ((tdt, ids), (F32, ids.int())):
        dtab, dpos = F.embedding_grad(g.to(DEV), width.to(DEV), V, scale=scale, positions=T if pos else 0, dtype=dt)
        r, m, n = embed_grad_ref(ids, g, V, scale)
        within(dtab, r, 1.01 * ((n + 1) * U * m + half(dt) * r.abs()), "d_table")
        if pos:
            r = g.double().sum(0)
            within(dpos, r, 1.01 * (B * U * g.double().abs().sum(0) + half(dt) * r.abs()), "d_pos")
        else:
            assert dpos is None


def test_embedding_ids_out_of_range_read_the_nearest_row(F):
    table = torch.arange(20, dtype=F32).reshape(5, 4)
    ids = torch.tensor([[-100, 0, 4, 5, 1 << 40]])
    assert torch.equal(F.embedding_forward(ids.to(DEV), table.to(DEV)).cpu(), table[torch.tensor([[0, 0, 4, 4, 4]])])
    d, _ = F.embedding_grad(torch.ones(1, 5, 4, device=DEV), ids.to(DEV), 5)
    assert torch.equal(d.cpu(), torch.tensor([2., 0, 0, 0, 3])[:, None].expand(5, 4))


def test_embedding_empty_and_strided(F):
    table = torch.randn(9, 24, generator=gen(1)).to(DEV)
    none = torch.zeros(0, 5, dtype=torch.long, device=DEV)
    assert F.embedding_forward(none, table).shape == (0, 5, 24)
    d, p = F.embedding_grad(torch.zeros(0, 5, 24, device=DEV), none, 9, positions=7)
    assert not d.any() and not p.any() and p.shape == (7, 24)
    # a column slice of a wider table, a transposed id matrix, a positional table with more rows than positions
    wide = torch.randn(9, 40, generator=gen(2)).to(DEV)
    ids = torch.randint(0, 9, (6, 4), generator=gen(3)).to(DEV)
    pos = torch.randn(11, 24, generator=gen(4)).to(DEV)
    got = F.embedding_forward(ids.t(), wide[:, 8:32], pos)
    assert torch.equal(got, wide[:, 8:32][ids.t()] + pos[:6])
    odd = F.embedding_forward(ids, wide[:, 1:25])  # rows that start off a 16-byte boundary
    assert torch.equal(odd, wide[:, 1:25][ids])
    g = torch.randn(4, 6, 24, generator=gen(5)).to(DEV)
    _, dp = F.embedding_grad(g.transpose(0, 1).contiguous().transpose(0, 1), ids.t(), 9, positions=11)
    assert dp.shape == (11, 24) and not dp[6:].any()
    within(dp[:6], g.double().cpu().sum(0), 5 * U * g.double().cpu().abs().sum(0))


def test_embedding_gradient_is_the_same_every_time(F):
    ids, _, _, g = embed_inputs(50, 400, 900, 256, BF16, BF16, False, seed=7, hot=0.5)
    ids, g = ids.to(DEV), g.to(DEV)
    first = F.embedding_grad(g, ids, 900, dtype=F32)[0]
    for _ in range(5):
        assert torch.equal(F.embedding_grad(g, ids, 900, dtype=F32)[0], first)


def test_embedding_autograd_and_refusals(F):
    ids, table, p, g = embed_inputs(3, 5, 11, 16, F32, F32, True, seed=9)
    table, p = table.to(DEV).requires_grad_(), p.to(DEV).requires_grad_()
    out = F.embedding(ids.to(DEV), table, p, scale=2.0)
    out.backward(g.to(DEV))
    r, m, n = embed_grad_ref(ids, g, 11, 2.0)
    within(table.grad, r, 1.01 * ((n + 1) * U * m + U * r.abs()))
    within(p.grad, g.double().sum(0), 4 * U * g.double().abs().sum(0))
    with pytest.raises(ValueError):
        F.embedding_forward(ids.to(DEV), table.detach().half())
    with pytest.raises(ValueError):
        F.embedding_forward(ids.float().to(DEV), table.detach())
    with pytest.raises(ValueError):
        F.embedding_forward(ids.to(DEV), table.detach(), p.detach()[:3])
    with pytest.raises(ValueError):
        F.embedding_grad(g.to(DEV)[:2], ids.to(DEV), 11)
    with pytest.raises(ValueError):
        F.embedding_grad(g.to(DEV), ids.to(DEV), 11, positions=2)


# ---- attention ----------------------------------------------------------------------------------------------------------
def attn_ref(q, k, v, g, causal, mask, scale, dtype):
    """Results in 64 bits and how far an fp32 evaluation (with probabilities rounded to `dtype`) may be from them.

    Scores: a sum of D products and two roundings of the scaled value, es; a probability, exp of a score less lse, is off by the
    errors of both (2 es) and of exp and the conversions (16 u); in bf16 by half a step more.  delta = g . o takes o as it was
    rounded.  Every further product adds the fp32 error of its own sum."""
    q, k, v, g = (t.double().transpose(1, 2) for t in (q, k, v, g))
    group = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    B, Hq, Tq, D = q.shape
    Tk = k.shape[2]
    hp, ho = (half(dtype) if dtype == BF16 else 0.0), half(dtype)
    see = torch.ones(B, 1, Tq, Tk, dtype=torch.bool)
    if causal:
        see = see & torch.ones(Tq, Tk, dtype=torch.bool).tril(Tk - Tq)
    if mask is not None:
        see = see & mask.bool()[:, None, None, :]
        hide = ~mask.bool()[:, None, :, None]
        k, v = k.masked_fill(hide, 0.0), v.masked_fill(hide, 0.0)
    s = q @ k.mT * scale
    mag = q.abs() @ k.abs().mT * abs(scale)
    es = ((D + 4) * U * mag).masked_fill(~see, 0.0).amax(-1, keepdim=True) if Tk else torch.zeros(B, Hq, Tq, 1).double()
    s = s.masked_fill(~see, -math.inf)
    lse = torch.logsumexp(s, -1)
    some = see.any(-1) if Tk else torch.zeros(B, 1, Tq, dtype=torch.bool)
    p = torch.exp(s - torch.where(some, lse, 0.0)[..., None])
    rel = 2 * es + (16 + Tk) * U + hp
    o = p @ v
    e_o = rel * (p @ v.abs()) + Tk * U * (p @ v.abs()) + ho * o.abs() + 1e-30
    e_lse = es[..., 0] + (8 + Tk) * U + 4 * U * torch.where(some, lse, 0.0).abs()
    dp = g @ v.mT
    delta = (g * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_dp = D * U * (g.abs() @ v.abs().mT)
    e_delta = (g.abs() * (e_o + D * U * o.abs())).sum(-1, keepdim=True)
    e_ds = ds.abs() * (rel + 4 * U) + p * (e_dp + e_delta)
    R = Tq * group
    dv, e_dv = p.mT @ g, (p * (rel + R * U)).mT @ g.abs()
    dq, e_dq = scale * ds @ k, abs(scale) * (e_ds + Tk * U * ds.abs()) @ k.abs()
    dk, e_dk = scale * ds.mT @ q, abs(scale) * (e_ds + R * U * ds.abs()).mT @ q.abs()
    fold = lambda t: t.reshape(B, Hq // group, group, Tk, D).sum(2)  # noqa: E731
    dk, e_dk, dv, e_dv = fold(dk), fold(e_dk), fold(dv), fold(e_dv)
    out = {}
    for name, t, e in (("o", o, e_o), ("dq", dq, e_dq), ("dk", dk, e_dk), ("dv", dv, e_dv)):
        out[name] = (t.transpose(1, 2), 1.01 * (e + ho * t.abs()).transpose(1, 2) + 1e-30)
    out["lse"] = (lse, 1.01 * e_lse)
    return out


def check_lse(got, ref, tol):
    got = got.double().cpu()
    none = ref == -math.inf
    assert torch.equal(got == -math.inf, none)
    within(got[~none], ref[~none], tol[~none], "lse")


def attn_inputs(B, Tq, Tk, Hq, Hkv, D, dtype, mask, seed=0):
    g = gen(seed)
    q, k, v, go = (torch.randn(*s, generator=g).to(dtype) for s in ((B, Tq, Hq, D), (B, Tk, Hkv, D), (B, Tk, Hkv, D), (B, Tq, Hq, D)))
    m = None
    if mask == "padded":
        n = torch.randint(0, Tk + 1, (B, 1), generator=g)
        n[0] = 0  # the first sequence has no key
        m = torch.arange(Tk) < n
    elif mask == "holes":
        m = torch.rand(B, Tk, generator=g) < 0.6
    return q, k, v, go, m


def attn_run(F, q, k, v, go, causal, m, scale=None):
    o, lse = F.attention_forward(q, k, v, causal=causal, key_mask=m, scale=scale)
    return {"o": o, "lse": lse, **dict(zip(("dq", "dk", "dv"), F.attention_grad(go, q, k, v, o, lse, causal=causal, key_mask=m, scale=scale)))}


def attn_check(got, ref):
    check_lse(got["lse"], *ref["lse"])
    for n in ("o", "dq", "dk", "dv"):
        within(got[n], *ref[n], n)


ATTN = [
    # B, Tq, Tk, Hq, Hkv, D, causal, mask
    (1, 1, 1, 1, 1, 32, False, None),
    (2, 1, 5, 4, 1, 64, True, None),
    (3, 29, 29, 2, 2, 256, True, None),
    (2, 29, 49, 2, 2, 256, False, "holes"),
    (2, 32, 64, 2, 1, 128, False, None),
    (2, 33, 65, 2, 2, 40, False, "padded"),
    (1, 129, 129, 2, 1, 72, True, "holes"),
    (3, 17, 200, 4, 2, 96, True, "padded"),
    (1, 200, 17, 2, 2, 64, True, None),       # more queries than keys: the first see none
    (1, 140, 300, 8, 1, 128, True, None),     # eight query heads to a key head
    (1, 1, 700, 8, 2, 128, True, "holes"),    # keys shared out over workgroups
    (2, 3, 1031, 2, 1, 256, False, "padded"),
    (1, 700, 40, 4, 2, 64, False, None),      # rows shared out over workgroups in the key gradients
    (1, 300, 300, 1, 1, 160, True, None),
    (4, 64, 128, 3, 3, 32, False, "padded"),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,Tq,Tk,Hq,Hkv,D,causal,mask", ATTN)
def test_attention(F, B, Tq, Tk, Hq, Hkv, D, causal, mask, dtype):
    q, k, v, go, m = attn_inputs(B, Tq, Tk, Hq, Hkv, D, dtype, mask)
    ref = attn_ref(q, k, v, go, causal, m, 1 / math.sqrt(D), dtype)
    got = attn_run(F, *(None if t is None else t.to(DEV) for t in (q, k, v, go)), causal, None if m is None else m.to(DEV))
    assert got["o"].dtype == dtype and got["dk"].dtype == dtype
    attn_check(got, ref)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_hidden_keys_may_hold_anything(F, dtype):
    q, k, v, go, m = attn_inputs(3, 50, 90, 4, 2, 64, dtype, "holes", seed=3)
    m[1] = False
    ref = attn_ref(q, k, v, go, False, m, 0.125, dtype)
    bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).min])
    fill = bad[torch.randint(0, 4, k.shape, generator=gen(4))].to(dtype)
    k, v = torch.where(m[:, :, None, None], k, fill), torch.where(m[:, :, None, None], v, fill)
    got = attn_run(F, q.to(DEV), k.to(DEV), v.to(DEV), go.to(DEV), False, m.to(DEV))
    attn_check(got, ref)
    assert not got["dk"][~m.to(DEV)].any() and not got["dv"][~m.to(DEV)].any() and not got["o"][1].any() and not got["dq"][1].any()


def test_attention_large_scores_and_scale(F):
    """Scores in the hundreds: the running maximum has to carry; the softmax is nearly one-hot."""
    q, k, v, go, _ = attn_inputs(1, 70, 150, 2, 2, 64, F32, None, seed=5)
    q = q * 8
    for scale in (1.0, -0.7):
        ref = attn_ref(q, k, v, go, False, None, float(torch.tensor(scale)), F32)
        attn_check(attn_run(F, *(t.to(DEV) for t in (q, k, v, go)), False, None, scale), ref)


def test_attention_strides(F):
    """Slices of one packed projection, heads before positions, a broadcast key, odd offsets, a strided mask."""
    g = gen(6)
    B, T, H, D = 2, 45, 2, 64
    packed = torch.randn(B, T, 3 * H * D, generator=g).to(BF16)
    q, k, v = (packed[..., i * H * D:(i + 1) * H * D].unflatten(-1, (H, D)) for i in range(3))
    go = torch.randn(B, H, T, D, generator=g).to(BF16).transpose(1, 2)
    ref = attn_ref(q, k, v, go, True, None, 0.125, BF16)
    dev = packed.to(DEV)
    dq, dk, dv = (dev[..., i * H * D:(i + 1) * H * D].unflatten(-1, (H, D)) for i in range(3))
    dgo = go.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    attn_check(attn_run(F, dq, dk, dv, dgo, True, None), ref)
    # off a 16-byte boundary: copied first
    flat = torch.randn(B * T * H * D + 1, generator=g).to(BF16)
    q1 = flat[1:].view(B, T, H, D)
    attn_check(attn_run(F, flat.to(DEV)[1:].view(B, T, H, D), dk, dv, dgo, True, None), attn_ref(q1, k, v, go, True, None, 0.125, BF16))
    # one key sequence for the whole batch; a mask whose rows are columns
    k0, v0 = k[:1].expand(B, T, H, D), v[:1].expand(B, T, H, D)
    m = torch.rand(T, B, generator=g) < 0.7
    got = attn_run(F, dq, dk[:1].expand(B, T, H, D), dv[:1].expand(B, T, H, D), dgo, False, m.to(DEV).t())
    attn_check(got, attn_ref(q, k0, v0, go, False, m.t(), 0.125, BF16))


def test_attention_empty(F):
    e = lambda *s: torch.zeros(*s, dtype=BF16, device=DEV)  # noqa: E731
    got = attn_run(F, e(2, 0, 2, 64), e(2, 5, 2, 64), e(2, 5, 2, 64), e(2, 0, 2, 64), False, None)
    assert got["o"].shape == (2, 0, 2, 64) and not got["dk"].any() and not got["dv"].any()
    got = attn_run(F, e(2, 3, 2, 64) + 1, e(2, 0, 2, 64), e(2, 0, 2, 64), e(2, 3, 2, 64) + 1, True, None)
    assert not got["o"].any() and (got["lse"] == -math.inf).all() and not got["dq"].any() and got["dk"].shape == (2, 0, 2, 64)
    got = attn_run(F, e(0, 3, 2, 64), e(0, 4, 2, 64), e(0, 4, 2, 64), e(0, 3, 2, 64), True, None)
    assert got["o"].shape == (0, 3, 2, 64) and got["dv"].shape == (0, 4, 2, 64)


def test_attention_is_the_same_every_time(F):
    q, k, v, go, _ = (None if t is None else t.to(DEV) for t in attn_inputs(1, 900, 300, 8, 2, 64, BF16, None, seed=8))
    first = attn_run(F, q, k, v, go, False, None)
    for _ in range(4):
        again = attn_run(F, q, k, v, go, False, None)
        assert all(torch.equal(again[n], first[n]) for n in first)


def test_attention_autograd_against_differences(F):
    """The gradient against central differences of the 64-bit definition, and what the differentiable call refuses."""
    q, k, v, go, m = attn_inputs(1, 6, 9, 2, 1, 32, F32, "holes", seed=10)
    m[:, :2] = True
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    F.attention(*leaves, causal=True, key_mask=m.to(DEV)).backward(go.to(DEV))
    scale = 1 / math.sqrt(32)

    def loss(q, k, v):
        return (attn_ref(q, k, v, go, True, m, scale, F32)["o"][0] * go.double()).sum()
    for leaf, i in zip(leaves, range(3)):
        direction = torch.randn(leaf.shape, generator=gen(11 + i), dtype=torch.float64)
        args = [q.double(), k.double(), v.double()]
        eps = 1e-5
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + eps * direction, args[i] - eps * direction
        diff = (loss(*hi) - loss(*lo)) / (2 * eps)  # off by eps^2 times a third derivative, about 1e-9 here
        got = (leaf.grad.double().cpu() * direction).sum()
        ref = attn_ref(q, k, v, go, True, m, scale, F32)[("dq", "dk", "dv")[i]]
        assert abs(got - diff) <= (ref[1] * direction.abs()).sum() + 1e-7
    with pytest.raises(ValueError):
        F.attention_forward(q.to(DEV), k.to(DEV), v.to(DEV, BF16))
    with pytest.raises(ValueError):
        F.attention_forward(q.to(DEV), k.to(DEV), v.to(DEV)[:, :3])
    with pytest.raises(ValueError):
        F.attention_forward(q.to(DEV), k.to(DEV), v.to(DEV), key_mask=m[:, :4].to(DEV))
    with pytest.raises(Exception, match="evenly"):
        F.attention_forward(torch.zeros(1, 2, 3, 32, device=DEV), torch.zeros(1, 2, 2, 32, device=DEV), torch.zeros(1, 2, 2, 32, device=DEV))
    with pytest.raises(Exception, match="columns"):
        F.attention_forward(*(torch.zeros(1, 2, 1, 260, device=DEV) for _ in range(3)))


# ---- vocabulary loss ----------------------------------------------------------------------------------------------------
def vocab_inputs(N, H, V, dtype, bias, seed=0, ignore_share=0.3):
    g = gen(seed)
    x, w = torch.randn(N, H, generator=g).to(dtype), (2.0 / math.sqrt(H) * torch.randn(V, H, generator=g)).to(dtype)
    b = 0.5 * torch.randn(V, generator=g) if bias else None
    t = torch.randint(0, V, (N,), generator=g)
    t = torch.where(torch.rand(N, generator=g) < ignore_share, torch.zeros_like(t), t)
    return x, w, b, t, torch.randn(N, generator=g)


def vocab_ref(x, w, b, t, a, ignore, dtype):
    """Results in 64 bits and bounds of an fp32 evaluation with d rounded to `dtype` for its products (bf16).

    A logit is a sum of H products and a bias, ez; lse is off by the largest ez and its own sum's error; a probability by both and
    by the roundings of the exponent (4 u |z|) and of exp (16 u)."""
    N, H = x.shape
    V = w.shape[0]
    hp, ho = (half(dtype) if dtype == BF16 else 0.0), half(dtype)
    X, W = x.double(), w.double()
    z = X @ W.T
    ez = (H + 3) * U * (X.abs() @ W.abs().T)
    if b is not None:
        z, ez = z + b.double(), ez + U * b.double().abs().masked_fill(b == -math.inf, 0.0)
    lse = torch.logsumexp(z, 1)
    fin = z.masked_fill(z == -math.inf, 0.0)
    e_lse = (ez + 4 * U * fin.abs()).amax(1) + (V + 16) * U + 2 * U * lse.abs()
    counted = (t >= 0) & (t < V)
    for i in ignore:
        counted &= t != i
    tt = t.clamp(0, V - 1)[:, None]
    loss = torch.where(counted, lse - z.gather(1, tt)[:, 0], 0.0)
    e_loss = torch.where(counted, e_lse + ez.gather(1, tt)[:, 0] + U * loss.abs() + U * fin.gather(1, tt)[:, 0].abs(), 0.0)
    p = torch.exp(z - lse[:, None])
    rel = ez + 4 * U * fin.abs() + e_lse[:, None] + 16 * U
    aw = torch.where(counted, a.double(), 0.0)[:, None]
    hot = torch.zeros_like(p).scatter_(1, tt, 1.0)
    d = aw * (p - hot)
    e_d = aw.abs() * p * rel + 3 * U * d.abs()
    e_dr = e_d + hp * (d.abs() + e_d)
    out = {"loss": (loss, 1.01 * e_loss + 1e-30), "lse": (lse, 1.01 * e_lse)}
    dx, dw, db = d @ W, d.T @ X, d.sum(0)
    out["dx"] = (dx, 1.01 * (e_dr @ W.abs() + V * U * (d.abs() @ W.abs()) + ho * dx.abs()) + 1e-30)
    out["dw"] = (dw, 1.01 * (e_dr.T @ X.abs() + N * U * (d.abs().T @ X.abs()) + ho * dw.abs()) + 1e-30)
    out["db"] = (db, 1.01 * (e_d.sum(0) + N * U * d.abs().sum(0) + U * db.abs()) + 1e-30) if b is not None else None
    return out


def vocab_run(F, x, w, b, t, a, ignore):
    loss, lse = F.vocab_loss_forward(x, w, t, bias=b, ignore=ignore)
    return {"loss": loss, "lse": lse, **dict(zip(("dx", "dw", "db"), F.vocab_loss_grad(a, x, w, t, lse, bias=b, ignore=ignore)))}


def vocab_check(got, ref):
    for n, r in ref.items():
        if r is None:
            assert got[n] is None
        else:
            within(got[n], *r, n)


def on(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


VOCAB = [
    # N, H, V, bias
    (1, 64, 300, True),
    (1, 8, 1, False),
    (24, 512, 3500, True),
    (130, 200, 129, True),
    (513, 64, 1031, False),
    (257, 300, 777, True),   # rows that are not whole 16 bytes in bf16
    (37, 33, 515, True),
    (200, 1024, 384, False),
    (700, 128, 128, True),
    (1, 2048, 5000, False),
    (1500, 136, 2000, True),  # gathered rows, k shared out over workgroups
    (600, 72, 9001, False),
    (300, 640, 257, True),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,H,V,bias", VOCAB)
def test_vocab_loss(F, N, H, V, bias, dtype):
    x, w, b, t, a = vocab_inputs(N, H, V, dtype, bias)
    got = vocab_run(F, *on(x, w, b, t, a), (0,))
    assert got["dx"].dtype == dtype and got["dw"].dtype == dtype
    vocab_check(got, vocab_ref(x, w, b, t, a, (0,), dtype))


def test_vocab_loss_in_pieces(F):
    """So many rows that d takes several pieces of the vocabulary; the gradients against sums over row blocks in 64 bits."""
    N, H, V = 100_000, 64, 3500
    x, w, b, t, a = vocab_inputs(N, H, V, BF16, True, seed=4)
    a = a / N
    X, Wm, B, T, A = on(x, w, b, t, a)
    got = vocab_run(F, X, Wm, B, T, A, (0,))
    ref = vocab_ref(x[:1000], w, b, t[:1000], a[:1000], (0,), BF16)
    for n in ("loss", "lse", "dx"):
        within(got[n][:1000], *ref[n], n)
    dw, db = torch.zeros(V, H, dtype=torch.float64, device=DEV), torch.zeros(V, dtype=torch.float64, device=DEV)
    mag_w, mag_b = torch.zeros_like(dw), torch.zeros_like(db)
    for lo in range(0, N, 10000):
        r = slice(lo, lo + 10000)
        z = X[r].double() @ Wm.double().T + B.double()
        d = torch.softmax(z, 1)
        d[torch.arange(d.shape[0]), T[r]] -= 1
        d *= (A[r].double() * (T[r] != 0))[:, None]
        dw += d.T @ X[r].double(); db += d.sum(0)
        mag_w += d.abs().T @ X[r].double().abs(); mag_b += d.abs().sum(0)
    # per element of d: a relative error below 2^-13 in fp32 (logits of up to 32, H = 64), then bf16 rounding for the products
    within(got["dw"], dw.cpu(), ((half(BF16) + 2.0 ** -13 + N * U) * mag_w + half(BF16) * dw.abs()).cpu(), "dw")
    within(got["db"], db.cpu(), ((2.0 ** -13 + N * U) * mag_b).cpu(), "db")


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_vocab_loss_masks(F, dtype):
    """Targets outside the vocabulary, several ignored words, words hidden by a bias of -infinity, rows that all do not count."""
    x, w, b, t, a = vocab_inputs(150, 96, 400, dtype, True, seed=2)
    t[3], t[7], t[11] = -100, 400, 1 << 40
    hide = torch.rand(400, generator=gen(3)) < 0.3
    hide[t.clamp(0, 399)] = False
    hide[128:256] = True  # whole tiles of hidden words
    t = torch.where((t >= 128) & (t < 256), torch.full_like(t, 2), t)
    hide[2] = False
    b = b.masked_fill(hide, -math.inf)
    got = vocab_run(F, *on(x, w, b, t, a), (0, 1, 5, -7))
    vocab_check(got, vocab_ref(x, w, b, t, a, (0, 1, 5, -7), dtype))
    assert not got["dw"][hide.to(DEV)].any() and got["loss"][3] == 0
    got = vocab_run(F, *on(x, w, b, torch.full_like(t, 5).int(), a), (5,))
    assert not got["loss"].any() and not got["dx"].any() and not got["dw"].any() and not got["db"].any() and torch.isfinite(got["lse"]).all()


@pytest.mark.parametrize("counted", [0, 1, 255, 256, 257, 511, 700])
def test_vocab_loss_counted_rows(F, counted):
    """So many of 700 rows count, anywhere among them: those alone go through the gradient's products."""
    x, w, b, _, a = vocab_inputs(700, 96, 600, BF16, True, seed=30)
    t = torch.zeros(700, dtype=torch.long)
    t[torch.randperm(700, generator=gen(31))[:counted]] = torch.randint(1, 600, (counted,), generator=gen(32))
    got = vocab_run(F, *on(x, w, b, t, a), (0,))
    vocab_check(got, vocab_ref(x, w, b, t, a, (0,), BF16))
    assert not got["dx"][(t == 0).to(DEV)].any()


def test_vocab_loss_strides_and_empty(F):
    x, w, b, t, a = vocab_inputs(60, 64, 200, BF16, True, seed=5)
    wide_x, wide_w = torch.randn(60, 104, generator=gen(6)).to(BF16), torch.randn(200, 80, generator=gen(7)).to(BF16)
    for lo_x, lo_w in ((8, 16), (3, 1)):  # in place, and off a 16-byte boundary
        wx, ww = wide_x[:, lo_x:lo_x + 64], wide_w[:, lo_w:lo_w + 64] * 0.2
        dev_w = (wide_w * 0.2).to(DEV)[:, lo_w:lo_w + 64]
        got = vocab_run(F, wide_x.to(DEV)[:, lo_x:lo_x + 64], dev_w, *on(b, t, a), (0,))
        vocab_check(got, vocab_ref(wx, ww, b, t, a, (0,), BF16))
    got = vocab_run(F, x.t().contiguous().to(DEV).t(), *on(w, b, t, a), (0,))  # columns first
    vocab_check(got, vocab_ref(x, w, b, t, a, (0,), BF16))
    got = vocab_run(F, *on(x[:0], w, b, t[:0], a[:0]), ())
    assert got["loss"].shape == (0,) and got["dx"].shape == (0, 64) and not got["dw"].any() and not got["db"].any()


def test_vocab_loss_is_the_same_every_time(F):
    args = on(*vocab_inputs(300, 256, 5000, BF16, True, seed=8))
    first = vocab_run(F, *args, (0,))
    for _ in range(4):
        again = vocab_run(F, *args, (0,))
        assert all(torch.equal(again[n], first[n]) for n in first)


def test_vocab_loss_autograd_against_differences(F):
    x, w, b, t, a = vocab_inputs(7, 16, 40, F32, True, seed=9)
    leaves = [v.to(DEV).requires_grad_() for v in (x, w, b)]
    (F.vocab_loss(leaves[0], leaves[1], t.to(DEV), bias=leaves[2], ignore=(0,)) * a.to(DEV)).sum().backward()
    ref = vocab_ref(x, w, b, t, a, (0,), F32)

    def loss(x, w, b):
        return (torch.nn.functional.cross_entropy(x @ w.T + b, t, reduction="none") * torch.where(t == 0, 0.0, a.double())).sum()
    for i, n in enumerate(("dx", "dw", "db")):
        args = [x.double(), w.double(), b.double()]
        direction = torch.randn(args[i].shape, generator=gen(20 + i), dtype=torch.float64)
        eps = 1e-5
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + eps * direction, args[i] - eps * direction
        diff = (loss(*hi) - loss(*lo)) / (2 * eps)  # off by eps^2 times a third derivative, about 1e-9 here
        got = (leaves[i].grad.double().cpu() * direction).sum()
        assert abs(got - diff) <= (ref[n][1] * direction.abs()).sum() + 1e-7
    # a mean over the counted rows: one scalar gradient for every row
    m = F.vocab_loss(leaves[0].detach().requires_grad_(), leaves[1], t.to(DEV), ignore=(0,)).sum()
    m.backward()
    with pytest.raises(ValueError):
        F.vocab_loss_forward(x.to(DEV), w.to(DEV, BF16), t.to(DEV))
    with pytest.raises(ValueError):
        F.vocab_loss_forward(x.to(DEV), w.to(DEV), t.to(DEV).float())
    with pytest.raises(ValueError):
        F.vocab_loss_forward(x.to(DEV), w.to(DEV), t.to(DEV), ignore=(1, 2, 3, 4, 5))
    with pytest.raises(ValueError):
        F.vocab_loss_forward(x.to(DEV), w.to(DEV), t.to(DEV), bias=b.to(DEV, BF16))
    with pytest.raises(ValueError):
        F.vocab_loss_grad(a.double().to(DEV), x.to(DEV), w.to(DEV), t.to(DEV), a.to(DEV))


# ---- all three in one step ----------------------------------------------------------------------------------------------
class Chain:
    """A one-layer decoder on the three operators: embedding + positions -> causal self-attention -> cross-attention to image
    tokens -> vocabulary loss, the projections left out; forward and all gradients by the plain calls."""

    def __init__(self, B=6, T=19, S=25, heads=2, D=64, V=700, dtype=BF16, seed=0):
        g = gen(seed)
        H = heads * D
        self.shape = (B, T, S, heads, D, V)
        self.ids = torch.randint(3, V, (B, T + 1), generator=g)
        n = torch.randint(3, T + 2, (B, 1), generator=g)
        self.ids = torch.where(torch.arange(T + 1) < n, self.ids, 0)
        self.table = (0.7 * torch.randn(V, H, generator=g)).to(dtype)
        self.pos = (0.7 * torch.randn(T, H, generator=g)).to(dtype)
        self.image = torch.randn(B, S, heads, D, generator=g).to(dtype)
        self.w = (0.3 * torch.randn(V, H, generator=g)).to(dtype)

    def cuda(self):
        for n in ("ids", "table", "pos", "image", "w"):
            setattr(self, n, getattr(self, n).to(DEV))
        return self

    def step(self, F):
        B, T, S, heads, D, V = self.shape
        ids, targets = self.ids[:, :-1], self.ids[:, 1:].reshape(-1)
        seen = ids != 0
        x = F.embedding_forward(ids, self.table, self.pos, scale=1.5)
        h = x.view(B, T, heads, D)
        o1, l1 = F.attention_forward(h, h, h, causal=True, key_mask=seen)
        o2, l2 = F.attention_forward(o1, self.image, self.image)
        y = o2.view(B * T, heads * D)
        loss, lse = F.vocab_loss_forward(y, self.w, targets, ignore=(0,))
        ones = torch.ones_like(loss)
        dy, dw, _ = F.vocab_loss_grad(ones, y, self.w, targets, lse, ignore=(0,))
        do1, dk2, dv2 = F.attention_grad(dy.view(B, T, heads, D), o1, self.image, self.image, o2, l2)
        dq, dk, dv = F.attention_grad(do1, h, h, h, o1, l1, causal=True, key_mask=seen)
        dx = (dq.float() + dk.float() + dv.float()).view(B, T, heads * D)
        dt, dp = F.embedding_grad(dx, ids, V, scale=1.5, positions=T, dtype=torch.float32)
        return {"loss": loss, "dw": dw, "dk2": dk2, "dv2": dv2, "dt": dt, "dp": dp}

    def reference(self):
        """The same in 64 bits by torch's automatic differentiation."""
        B, T, S, heads, D, V = self.shape
        table, pos, w = (t.double().requires_grad_() for t in (self.table, self.pos, self.w))
        k2, v2 = (self.image.double().requires_grad_() for _ in range(2))
        ids, targets = self.ids[:, :-1], self.ids[:, 1:].reshape(-1)
        h = (1.5 * table[ids] + pos).view(B, T, heads, D).transpose(1, 2)

        def attend(q, k, v, see):
            s = (q @ k.mT / math.sqrt(D)).masked_fill(~see, -1e300)
            return torch.softmax(s, -1) * see.any(-1, keepdim=True) @ v
        see = torch.ones(T, T, dtype=torch.bool).tril() & (ids != 0)[:, None, None, :]
        o1 = attend(h, h, h, see)
        o2 = attend(o1, k2.transpose(1, 2), v2.transpose(1, 2), torch.ones(T, S, dtype=torch.bool))
        z = o2.transpose(1, 2).reshape(B * T, heads * D) @ w.T
        loss = torch.nn.functional.cross_entropy(z, targets, reduction="none", ignore_index=0)
        loss.sum().backward()
        return {"loss": loss.detach(), "dw": w.grad, "dk2": k2.grad, "dv2": v2.grad, "dt": table.grad, "dp": pos.grad}


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_chain(F, dtype):
    """Rounded intermediate tensors (eight roundings to `dtype` between the table and the gradients) and fp32 sums of a few
    thousand terms: relative error in norm below 16 half steps, plus 2^-14 for the sums."""
    c = Chain(dtype=dtype)
    ref = c.reference()
    got = c.cuda().step(F)
    for n, r in ref.items():
        err = (got[n].double().cpu() - r).norm() / r.norm()
        assert err <= 16 * half(dtype) + 2.0 ** -14, (n, float(err))


def test_chain_in_a_graph(F):
    """Captured once, replayed with other inputs between eager steps: every replay equals the eager step, bit for bit."""
    c = Chain(seed=1).cuda()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        c.step(F)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = c.step(F)
    for k in range(4):
        other = Chain(seed=10 + k).cuda()
        for n in ("ids", "table", "pos", "image", "w"):
            getattr(c, n).copy_(getattr(other, n))
        graph.replay()
        eager = other.step(F)
        torch.cuda.synchronize()
        for n in eager:
            assert torch.equal(held[n], eager[n]), (k, n)


def test_chain_on_two_streams(F):
    """Two steps in flight at once, each on its own stream, against the same steps one after another."""
    cs = [Chain(seed=s, B=9, T=60).cuda() for s in (5, 6)]
    alone = [c.step(F) for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    for _ in range(3):
        got = []
        for c, s in zip(cs, streams):
            with torch.cuda.stream(s):
                got.append(c.step(F))
        torch.cuda.synchronize()
        for g, a in zip(got, alone):
            for n in a:
                assert torch.equal(g[n], a[n]), n
