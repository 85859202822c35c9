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


def attn_desc(L, **kw):
    d = L.AttnSeqDesc()
    for n in ("q", "k", "v", "o", "lse", "grad_o", "dq", "dk", "dv", "workspace"):
        setattr(d, n, P)
    for n in ("q_stride", "k_stride", "v_stride", "o_stride", "g_stride"):
        for i, v in enumerate((1 << 20, 64, 32)):
            getattr(d, n)[i] = v
    d.dtype, d.B, d.Tq, d.Tk, d.Hq, d.Hkv, d.D, d.scale = L.BF16, 2, 3, 5, 2, 1, 32, 0.2
    d.workspace_bytes = 1 << 30
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_attn_seq_refuses(L):
    import ctypes as C
    calls = [L.lib.mic_attn_seq, L.lib.mic_attn_seq_grad]
    for f in calls:
        refused(L, f(None, None), b"null descriptor")
        refused(L, f(C.byref(attn_desc(L, dtype=3)), None), b"dtype")
        for kw in (dict(B=-1), dict(Tq=-1), dict(Tk=-2), dict(Hq=0), dict(Hkv=0), dict(D=0)):
            refused(L, f(C.byref(attn_desc(L, **kw)), None), b"bad sizes")
        refused(L, f(C.byref(attn_desc(L, Hq=3, Hkv=2)), None), b"evenly")
        refused(L, f(C.byref(attn_desc(L, D=264)), None), b"columns")
        refused(L, f(C.byref(attn_desc(L, D=36)), None), b"columns")
        assert L.lib.mic_attn_seq_workspace_bytes(C.byref(attn_desc(L, dtype=L.F32, D=36)), 0) >= 0  # 36 floats are whole 16 bytes
        refused(L, f(C.byref(attn_desc(L, B=1 << 20, Tq=1 << 20)), None), b"too many rows")
        refused(L, f(C.byref(attn_desc(L, Tq=1 << 30)), None), b"too many rows")
        for n in ("q", "k", "v", "o", "lse"):
            refused(L, f(C.byref(attn_desc(L, **{n: None})), None), b"null pointer")
        refused(L, f(C.byref(attn_desc(L, k=P + 8)), None), b"aligned")
        for s in ("q_stride", "k_stride", "v_stride", "o_stride"):
            d = attn_desc(L)
            getattr(d, s)[1] = 33
            refused(L, f(C.byref(d), None), b"stride")
            getattr(d, s)[1] = -64
            refused(L, f(C.byref(d), None), b"stride")
        for i, far in ((1, (1 << 23) + 8), (2, 1 << 29)):  # 64 positions, the heads of one, beyond 1 GiB
            d = attn_desc(L)
            d.k_stride[i] = far if i == 1 else far + 8
            refused(L, f(C.byref(d), None), b"too large")
    for n in ("dq", "dk", "dv"):
        refused(L, L.lib.mic_attn_seq_grad(C.byref(attn_desc(L, **{n: None})), None), b"null pointer")
    refused(L, L.lib.mic_attn_seq_grad(C.byref(attn_desc(L, dv=P + 4)), None), b"aligned")
    d = attn_desc(L)
    need = L.lib.mic_attn_seq_workspace_bytes(C.byref(d), 1)
    assert need >= 2 * 2 * 3 * 4
    for kw in (dict(workspace_bytes=need - 1), dict(workspace=None), dict(workspace=P + 8)):
        refused(L, L.lib.mic_attn_seq_grad(C.byref(attn_desc(L, **kw)), None), b"workspace")
    long = dict(B=1, Tq=1, Tk=8192)  # one row over many keys: shared out, which needs scratch
    need = L.lib.mic_attn_seq_workspace_bytes(C.byref(attn_desc(L, **long)), 0)
    assert need > 0
    refused(L, L.lib.mic_attn_seq(C.byref(attn_desc(L, workspace_bytes=need - 1, **long)), None), b"workspace")
    assert L.lib.mic_attn_seq(C.byref(attn_desc(L, B=0)), None) == 0 and L.lib.mic_attn_seq_grad(C.byref(attn_desc(L, B=0)), None) == 0
    refused(L, L.lib.mic_attn_seq_workspace_bytes(C.byref(attn_desc(L, D=300)), 0), b"columns")


def vocab_desc(L, **kw):
    d = L.VocabLossDesc()
    for n in ("x", "w", "bias", "targets", "loss", "lse", "grad_rows", "dx", "dw", "db", "workspace"):
        setattr(d, n, P)
    d.ld_x = d.ld_w = 64
    d.dtype, d.N, d.H, d.V, d.target_bits, d.n_ignore, d.workspace_bytes = L.BF16, 10, 64, 300, 64, 1, 1 << 40
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_vocab_loss_refuses(L):
    import ctypes as C
    for f in (L.lib.mic_vocab_loss, L.lib.mic_vocab_loss_grad):
        refused(L, f(None, None), b"null descriptor")
        refused(L, f(C.byref(vocab_desc(L, dtype=2)), None), b"dtype")
        for kw in (dict(N=-1), dict(H=0), dict(V=0)):
            refused(L, f(C.byref(vocab_desc(L, **kw)), None), b"bad sizes")
        refused(L, f(C.byref(vocab_desc(L, N=1 << 30)), None), b"range")
        refused(L, f(C.byref(vocab_desc(L, N=1 << 29, V=1 << 29)), None), b"range")
        refused(L, f(C.byref(vocab_desc(L, target_bits=16)), None), b"bits")
        refused(L, f(C.byref(vocab_desc(L, n_ignore=5)), None), b"ignored")
        refused(L, f(C.byref(vocab_desc(L, n_ignore=-1)), None), b"ignored")
        refused(L, f(C.byref(vocab_desc(L, ld_x=63)), None), b"row stride")
        refused(L, f(C.byref(vocab_desc(L, ld_w=0)), None), b"row stride")
        for n in ("x", "w", "targets", "lse"):
            refused(L, f(C.byref(vocab_desc(L, **{n: None})), None), b"null pointer")
    need = L.lib.mic_vocab_loss_workspace_bytes(C.byref(vocab_desc(L)), 0)
    assert need > 0
    refused(L, L.lib.mic_vocab_loss(C.byref(vocab_desc(L, workspace_bytes=need - 1)), None), b"workspace")
    refused(L, L.lib.mic_vocab_loss(C.byref(vocab_desc(L, workspace=P + 8)), None), b"workspace")
    refused(L, L.lib.mic_vocab_loss(C.byref(vocab_desc(L, loss=None)), None), b"null pointer")
    for n in ("grad_rows", "dx", "dw"):
        refused(L, L.lib.mic_vocab_loss_grad(C.byref(vocab_desc(L, **{n: None})), None), b"null pointer")
    for n in ("dx", "dw", "db"):
        refused(L, L.lib.mic_vocab_loss_grad(C.byref(vocab_desc(L, **{n: P + 4})), None), b"aligned")
    need = L.lib.mic_vocab_loss_workspace_bytes(C.byref(vocab_desc(L)), 1)
    refused(L, L.lib.mic_vocab_loss_grad(C.byref(vocab_desc(L, workspace_bytes=need - 1)), None), b"workspace")
    assert L.lib.mic_vocab_loss(C.byref(vocab_desc(L, N=0, x=None, targets=None, lse=None)), None) == 0
    refused(L, L.lib.mic_vocab_loss_workspace_bytes(C.byref(vocab_desc(L, V=-5)), 1), b"bad sizes")
    assert L.lib.mic_vocab_loss_workspace_bytes(C.byref(vocab_desc(L, N=0)), 0) == 0
    assert L.lib.mic_vocab_loss_workspace_bytes(C.byref(vocab_desc(L, N=0)), 1) == 0


def test_workspace_sizes_of_empty_calls(L):
    import ctypes as C
    assert L.lib.mic_embed_grad_workspace_bytes(0, 1, 8, 5, 1) >= 0
    for kw in (dict(B=0), dict(Tq=0), dict(Tk=0), dict(Tq=0, Tk=0)):
        for grad in (0, 1):
            assert L.lib.mic_attn_seq_workspace_bytes(C.byref(attn_desc(L, **kw)), grad) >= 0


def test_packed_descriptors_match_the_header(L, F):
    """The Python layer packs the descriptors in one go: every field has to land where the header has it."""
    import ctypes as C
    import os
    import subprocess
    import tempfile
    n = len(L.AttnSeqDesc._fields_)
    assert F._ATTN_PACK.size == C.sizeof(L.AttnSeqDesc) and F._VOCAB_PACK.size == C.sizeof(L.VocabLossDesc) and n == 27
    d = L.AttnSeqDesc.from_buffer_copy(F._ATTN_PACK.pack(*range(1, 35), 0.5, 35, 36))
    assert [getattr(d, f) for f in ("q", "k", "v", "o", "lse", "key_mask", "grad_o", "dq", "dk", "dv")] == list(range(1, 11))
    assert [x for f in ("q_stride", "k_stride", "v_stride", "o_stride", "g_stride") for x in getattr(d, f)] == list(range(11, 26))
    assert [getattr(d, f) for f in ("mask_stride", "dtype", "B", "Tq", "Tk", "Hq", "Hkv", "D", "causal", "scale", "workspace", "workspace_bytes")] == \
        [26, 27, 28, 29, 30, 31, 32, 33, 34, 0.5, 35, 36]
    d = L.VocabLossDesc.from_buffer_copy(F._VOCAB_PACK.pack(*range(1, 25)))
    assert [getattr(d, f) for f, _ in L.VocabLossDesc._fields_ if f != "ignore"] == [*range(1, 19), 23, 24] and list(d.ignore) == [19, 20, 21, 22]
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = """#include <stdio.h>
#include <stddef.h>
#include "mic_hip.h"
int main(void) { printf("%zu %zu %zu %zu %zu %zu\\n", sizeof(mic_attn_seq_desc), offsetof(mic_attn_seq_desc, mask_stride), offsetof(mic_attn_seq_desc, workspace),
  sizeof(mic_vocab_loss_desc), offsetof(mic_vocab_loss_desc, n_ignore), offsetof(mic_vocab_loss_desc, workspace)); return 0; }"""
    with tempfile.TemporaryDirectory() as tmp:
        c, exe = os.path.join(tmp, "t.c"), os.path.join(tmp, "t")
        open(c, "w").write(src)
        subprocess.run(["gcc", "-I", os.path.join(root, "include"), c, "-o", exe], check=True)
        got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(L.AttnSeqDesc), L.AttnSeqDesc.mask_stride.offset, L.AttnSeqDesc.workspace.offset,
                   C.sizeof(L.VocabLossDesc), L.VocabLossDesc.n_ignore.offset, L.VocabLossDesc.workspace.offset]


def test_sizes_beyond_a_launch_are_refused(L):
    """What would need 2^32 threads or more in one launch, or more scratch than 64 bits of bytes tell."""
    import ctypes as C
    assert L.lib.mic_embed_grad_workspace_bytes(1 << 16, 1 << 16, 1 << 14, 100, 1) >= 0
    assert L.lib.mic_embed_grad_workspace_bytes(1 << 16, 1 << 16, 1 << 15, 100, 1) < 0
    assert L.lib.mic_embed_grad_workspace_bytes(8, 8, (1 << 20) + 8, 100, 0) < 0
    d = attn_desc(L, B=1, Tq=1, Hq=(1 << 20) + 2, Hkv=1)
    refused(L, L.lib.mic_attn_seq(C.byref(d), None), b"too many rows")
    d = attn_desc(L, B=1 << 22, Tq=1)
    refused(L, L.lib.mic_attn_seq(C.byref(d), None), b"too many rows")
    for N, H, V in ((1 << 26, 8, 8), (8, 1 << 28, 8), (8, 8, 1 << 28), (1 << 24, 1 << 10, 8), (8, 1 << 10, 1 << 24), (1 << 20, 8, 1 << 20)):
        v = L.VocabLossDesc()
        v.dtype, v.N, v.H, v.V, v.target_bits, v.ld_x, v.ld_w = L.BF16, N, H, V, 32, H, H
        for grad in (0, 1):
            assert L.lib.mic_vocab_loss_workspace_bytes(C.byref(v), grad) == -1 and b"sizes out of range" in L.lib.mic_last_error()
    v.N, v.H, v.V, v.ld_x, v.ld_w = 1 << 17, 1 << 10, 1 << 17, 1 << 10, 1 << 10
    assert L.lib.mic_vocab_loss_workspace_bytes(C.byref(v), 1) < 16 << 30  # d and the partial dx share a few GiB


def test_vocab_loss_of_many_small_tiles_takes_larger_ones(L):
    """2^36 logits on tiles of 64 x 64 would be a launch of 2^32 threads; a row's statistics are kept for every half tile of columns, so
    the scratch tells the tile."""
    import ctypes as C
    v = L.VocabLossDesc()
    v.V, v.target_bits = 4096, 32
    for dtype, H in ((L.BF16, 8), (L.F32, 64)):
        v.dtype, v.H, v.ld_x, v.ld_w = dtype, H, H, H
        for N, half_tile in (((1 << 24) - 64, 32), (1 << 24, 64), ((1 << 24) + 5, 64)):
            v.N = N
            parts = v.V // half_tile
            need = L.lib.mic_vocab_loss_workspace_bytes(C.byref(v), 0)
            assert abs(need - N * (parts * 8 + 4)) <= 1024, (dtype, N, need)


def test_vocab_loss_gradient_scratch(L):
    """Beside the gathered rows, a piece of d and the column sums: per piece a copy of dx and the partial tiles of one round of workgroups
    (256 of 256 x 256, 512 of 128 x 128 or 1024 of 64 x 64) at most."""
    import ctypes as C
    v = L.VocabLossDesc()
    v.target_bits, v.db = 64, P
    for dtype, N, H, V, pieces, width, tile in ((L.BF16, 7424, 512, 3500, 1, 3500, 256), (L.BF16, 256, 2048, 65536, 1, 65536, 256),
                                                (L.BF16, 4096, 2048, 32000, 1, 32000, 256), (L.BF16, 8192, 2048, 65536, 4, 16384, 256),
                                                (L.F32, 7424, 512, 3500, 1, 3500, 64), (L.F32, 1111, 300, 10007, 1, 10007, 64),
                                                (L.BF16, 100, 1024, 70000, 1, 70000, 128), (L.BF16, 24, 512, 32000, 1, 32000, 64)):
        v.dtype, v.N, v.H, v.V, v.ld_x, v.ld_w = dtype, N, H, V, H, H
        size = 4 if dtype == L.F32 else 2
        round_ = {256: 256, 128: 512, 64: 1024}[tile] * tile * tile
        most = N * H * size + N * (width + 8) * size + pieces * (N * H + round_) * 4 + -(-N // tile) * 2 * width * 4 + 16 * N + (1 << 16)
        assert L.lib.mic_vocab_loss_workspace_bytes(C.byref(v), 1) <= most, (dtype, N, H, V)


def test_vocab_loss_limits_are_those_of_the_header(L):
    """Each size alone at its limit, and one step of 64 beyond it."""
    import ctypes as C
    v = L.VocabLossDesc()
    v.dtype, v.target_bits = L.BF16, 64
    edge = lambda units: (units - 2) * 64 + 63  # noqa: E731  (the largest size of so many units)
    for N, H, V in ((edge(1 << 19), 8, 8), (8, edge((1 << 20) - 1), 8), (8, 8, edge((1 << 20) - 1)), (edge(1 << 14), 8, edge((1 << 11) - 1)),
                    (edge(1 << 11), edge((1 << 10) - 1), 8)):
        for k in range(4):
            sizes = [N, H, V]
            if k:
                sizes[k - 1] += 64
            v.N, v.H, v.V, v.ld_x, v.ld_w = *sizes, sizes[1], sizes[1]
            n, h, w = (s // 64 + 2 for s in sizes)
            fits = n <= 1 << 19 and h <= 1 << 21 and w <= 1 << 21 and n * w < 1 << 25 and n * h < 1 << 21 and w * h < 1 << 21
            assert k or fits
            for grad in (0, 1):
                assert (L.lib.mic_vocab_loss_workspace_bytes(C.byref(v), grad) >= 0) == fits, sizes
