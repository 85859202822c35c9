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
