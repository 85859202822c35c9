"""What the teacher-forced operators refuse, checked without a GPU: the library validates before its first HIP call, the
Python layer before it touches the library."""
import pytest
import torch


@pytest.fixture(scope="module")
def L():
    import image_captioning_amd as m
    return m._lib


@pytest.fixture(scope="module")
def F():
    import image_captioning_amd as m
    return m.functional


P = 4096  # a non-null, 16-byte aligned address that a refused call never reads


def refused(L, rc, text):
    assert rc == -1
    assert text in L.lib.mic_last_error(), L.lib.mic_last_error()


def test_embed_rows_refuses(L):
    f = L.lib.mic_embed_rows
    good = dict(ids=P, bits=64, table=P, ld=8, pos=None, ldp=0, out=P, td=L.F32, od=L.BF16, scale=1.0, n=4, T=2, H=8, V=5)

    def call(**kw):
        a = {**good, **kw}
        return f(a["ids"], a["bits"], a["table"], a["ld"], a["pos"], a["ldp"], a["out"], a["td"], a["od"], a["scale"], a["n"], a["T"], a["H"],
                 a["V"], None)
    for kw in (dict(n=-1), dict(n=1 << 31), dict(T=0), dict(H=0), dict(V=0)):
        refused(L, call(**kw), b"bad sizes")
    refused(L, call(bits=16), b"bits")
    refused(L, call(td=7), b"dtype")
    refused(L, call(od=-1), b"dtype")
    refused(L, call(ld=7), b"row stride")
    refused(L, call(pos=P, ldp=3), b"row stride")
    for k in ("ids", "table", "out"):
        refused(L, call(**{k: None}), b"null pointer")
    assert call(n=0, ids=None, table=None, out=None) == 0  # nothing to do


def test_embed_grad_refuses(L):
    ws = L.lib.mic_embed_grad_workspace_bytes
    assert ws(6, 3, 8, 5, 1) > 0 and ws(6, 3, 8, 5, 0) > 0
    for a in ((-1, 3, 8, 5, 0), (1 << 30, 3, 8, 5, 0), (6, 0, 8, 5, 0), (6, 3, 0, 5, 0), (6, 3, 8, 0, 0), (7, 3, 8, 5, 1)):
        assert ws(*a) == -1, a
    need = ws(6, 3, 8, 5, 1)
    good = dict(ids=P, bits=64, g=P, dt=P, dp=P, gd=L.BF16, od=L.F32, n=6, T=3, H=8, V=5, ws=P, size=need)

    def call(**kw):
        a = {**good, **kw}
        return L.lib.mic_embed_grad(a["ids"], a["bits"], a["g"], a["dt"], a["dp"], a["gd"], a["od"], 1.0, a["n"], a["T"], a["H"], a["V"], a["ws"],
                                    a["size"], None)
    for kw in (dict(n=-1), dict(n=1 << 30), dict(T=0), dict(H=0), dict(V=0)):
        refused(L, call(**kw), b"bad sizes")
    refused(L, call(bits=8), b"bits")
    refused(L, call(gd=9), b"dtype")
    refused(L, call(od=9), b"dtype")
    refused(L, call(n=7), b"whole sequences")
    for k in ("ids", "g", "dt"):
        refused(L, call(**{k: None}), b"null pointer")
    refused(L, call(size=need - 1), b"workspace")
    refused(L, call(ws=None), b"workspace")
    refused(L, call(ws=P + 4), b"aligned")


def test_python_layer_refuses_cpu_tensors(F):
    with pytest.raises(ValueError, match="HIP device"):
        F.embedding_forward(torch.zeros(2, 3, dtype=torch.long), torch.zeros(5, 8))
    with pytest.raises(ValueError, match="HIP device"):
        F.embedding_grad(torch.zeros(2, 3, 8), torch.zeros(2, 3, dtype=torch.long), 5)
