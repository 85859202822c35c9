"""Teacher-forced operators of the caption decoders on whole sequences, with their gradients.

The decode path takes one position at a time and needs no gradient; a training or scoring step (train.py:163-262 of the
reference) takes whole captions.  Each operator comes as a pair of plain calls, ``*_forward`` and ``*_grad``, that enqueue
kernels on the current stream of the tensors' device and return new tensors, and as one differentiable call for
``torch.autograd`` built on the pair: ``embedding``, ``attention``, ``vocab_loss``.

Tensors live on one HIP device, fp32 or bf16.  Nothing synchronises; every call may be captured into a HIP graph (workspaces
come from torch's allocator, which gives a captured graph a pool of its own).  Refused arguments raise ``ValueError`` (shapes,
types, devices) or ``_lib.MicError`` (what the library refuses).
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import torch

from . import _lib as L

__all__ = ["embedding", "embedding_forward", "embedding_grad", "attention", "attention_forward", "attention_grad",
           "vocab_loss", "vocab_loss_forward", "vocab_loss_grad"]


def _device(name: str, *tensors) -> torch.device:
    """The one HIP device all given tensors (None is skipped) live on."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{name}: expected tensors, got {type(t).__name__}")
        if t.device.type != "cuda":
            raise ValueError(f"{name}: tensors must be on a HIP device, got one on {t.device}")
        if dev is not None and t.device != dev:
            raise ValueError(f"{name}: tensors are on {dev} and {t.device}")
        dev = t.device
    return dev


def _need(ok: bool, name: str, what: str) -> None:
    if not ok:
        raise ValueError(f"{name}: {what}")


def _float_code(name: str, what: str, dtype) -> int:
    if dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"{name}: {what} must be float32 or bfloat16, got {dtype}")
    return L.F32 if dtype == torch.float32 else L.BF16


def _workspace(name: str, size: int, dev) -> torch.Tensor:
    if size < 0:
        raise ValueError(f"{name}: sizes out of range")
    return torch.empty(size, dtype=torch.uint8, device=dev)


def _ids(name: str, what: str, t: torch.Tensor) -> torch.Tensor:
    _need(t.dtype in (torch.int32, torch.int64), name, f"{what} must be int32 or int64, got {t.dtype}")
    return t.contiguous()


def _stream(dev) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


# ---- embedding --------------------------------------------------------------------------------------------------------
def embedding_forward(ids: torch.Tensor, table: torch.Tensor, pos: Optional[torch.Tensor] = None, *, scale: float = 1.0,
                      dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``scale * table[ids] + pos`` rounded once to ``dtype`` (the table's by default); models/transformer.py:44-50.

    ids (..., T) int32 / int64; table (vocab, H); pos (at least T rows, H) in the table's dtype, row t added at position t of the
    last dimension of ids.  Ids outside the vocabulary read its nearest row.  Returns (..., T, H)."""
    name = "embedding_forward"
    dev = _device(name, ids, table, pos)
    _need(table.dim() == 2 and table.shape[0] > 0 and table.shape[1] > 0, name, f"table must be (vocab, H), got {tuple(table.shape)}")
    _need(ids.dim() >= 1, name, "ids need at least one dimension")
    H, T = table.shape[1], ids.shape[-1]
    code = _float_code(name, "the table", table.dtype)
    out_dtype = dtype if dtype is not None else table.dtype
    out_code = _float_code(name, "the output", out_dtype)
    if pos is not None:
        _need(pos.dim() == 2 and pos.shape[1] == H and pos.shape[0] >= T and pos.dtype == table.dtype, name,
              f"pos must be (>= {T}, {H}) of {table.dtype}, got {tuple(pos.shape)} of {pos.dtype}")
        pos = pos if pos.stride(1) == 1 and pos.stride(0) >= H else pos.contiguous()
    table = table if table.stride(1) == 1 and table.stride(0) >= H else table.contiguous()
    ids = _ids(name, "ids", ids)
    out = torch.empty(*ids.shape, H, dtype=out_dtype, device=dev)
    if ids.numel() == 0:
        return out
    with torch.cuda.device(dev):
        L.check(L.lib.mic_embed_rows(ids.data_ptr(), 64 if ids.dtype == torch.int64 else 32, table.data_ptr(), table.stride(0), L.ptr(pos),
                                     pos.stride(0) if pos is not None else 0, out.data_ptr(), code, out_code, scale, ids.numel(), T, H,
                                     table.shape[0], _stream(dev)), "mic_embed_rows")
    return out


def embedding_grad(grad: torch.Tensor, ids: torch.Tensor, vocab: int, *, scale: float = 1.0, positions: int = 0,
                   dtype: Optional[torch.dtype] = None):
    """Gradients of ``embedding_forward``: (d_table (vocab, H), d_pos (positions, H) or None), rounded once to ``dtype`` (grad's by
    default).  grad (..., T, H) is the gradient of the output; positions is the row count of the positional table, 0 for none.
    Sums run in fp32 over the tokens sorted by word: the same inputs give the same bits."""
    name = "embedding_grad"
    dev = _device(name, grad, ids)
    _need(ids.dim() >= 1 and grad.shape[:-1] == ids.shape and grad.dim() == ids.dim() + 1, name,
          f"grad {tuple(grad.shape)} does not fit ids {tuple(ids.shape)}")
    H, T, n = grad.shape[-1], ids.shape[-1], ids.numel()
    _need(H > 0 and vocab > 0, name, f"bad sizes H={H} vocab={vocab}")
    _need(positions == 0 or positions >= T, name, f"{positions} positions for sequences of {T}")
    code = _float_code(name, "grad", grad.dtype)
    out_dtype = dtype if dtype is not None else grad.dtype
    out_code = _float_code(name, "the gradients", out_dtype)
    ids, grad = _ids(name, "ids", ids), grad.contiguous()
    d_table = torch.empty(vocab, H, dtype=out_dtype, device=dev)
    d_pos = None
    if positions:
        d_pos = torch.empty(positions, H, dtype=out_dtype, device=dev)
        if positions > T:
            d_pos[T:].zero_()
    T = max(T, 1)
    with torch.cuda.device(dev):
        ws = _workspace(name, int(L.lib.mic_embed_grad_workspace_bytes(n, T, H, vocab, int(bool(positions)))), dev)
        L.check(L.lib.mic_embed_grad(ids.data_ptr(), 64 if ids.dtype == torch.int64 else 32, grad.data_ptr(), d_table.data_ptr(), L.ptr(d_pos),
                                     code, out_code, scale, n, T, H, vocab, ws.data_ptr(), ws.numel(), _stream(dev)), "mic_embed_grad")
    return d_table, d_pos


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, pos, scale, dtype):
        ctx.save_for_backward(ids)
        ctx.meta = (table.shape[0], scale, 0 if pos is None else pos.shape[0], table.dtype)
        return embedding_forward(ids, table, pos, scale=scale, dtype=dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        vocab, scale, positions, dtype = ctx.meta
        d_table, d_pos = embedding_grad(grad, ids, vocab, scale=scale, positions=positions if ctx.needs_input_grad[2] else 0, dtype=dtype)
        return None, d_table, d_pos, None, None


def embedding(ids, table, pos=None, *, scale: float = 1.0, dtype=None) -> torch.Tensor:
    """``embedding_forward`` that ``torch.autograd`` can differentiate with respect to ``table`` and ``pos``."""
    return _Embedding.apply(ids, table, pos, scale, dtype)


# ---- attention --------------------------------------------------------------------------------------------------------
def _heads(t: torch.Tensor) -> torch.Tensor:
    """The tensor itself where the kernels can read it in place (columns consecutive, everything on 16-byte boundaries)."""
    e = 16 // t.element_size()
    if t.data_ptr() % 16 == 0 and (t.stride(3) == 1 or t.shape[3] == 1) and all(s % e == 0 for s in _strides(t)):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(t: torch.Tensor):
    """Strides of (batch, position, head); a dimension of one entry has none to speak of."""
    return (C.c_int64 * 3)(*(t.stride(i) if t.shape[i] > 1 else 0 for i in range(3)))


def _attn_desc(name, q, k, v, causal, key_mask, scale):
    dev = _device(name, q, k, v, key_mask)
    _need(q.dim() == 4 and k.dim() == 4 and v.dim() == 4, name, "q, k and v must be (batch, positions, heads, columns)")
    B, Tq, Hq, D = q.shape
    Tk, Hkv = k.shape[1], k.shape[2]
    _need(k.shape == v.shape and k.shape[0] == B and k.shape[3] == D and Hq > 0 and Hkv > 0 and D > 0, name,
          f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit")
    _need(k.dtype == q.dtype and v.dtype == q.dtype, name, f"q, k and v are {q.dtype}, {k.dtype} and {v.dtype}")
    d = L.AttnSeqDesc()
    d.dtype = _float_code(name, "q", q.dtype)
    q, k, v = _heads(q), _heads(k), _heads(v)
    if key_mask is not None:
        _need(key_mask.dtype in (torch.bool, torch.uint8) and key_mask.shape == (B, Tk), name,
              f"key_mask must be bool ({B}, {Tk}), got {key_mask.dtype} {tuple(key_mask.shape)}")
        if Tk > 1 and key_mask.stride(1) != 1:
            key_mask = key_mask.contiguous()
        d.key_mask, d.mask_stride = key_mask.data_ptr(), key_mask.stride(0)
    d.q, d.k, d.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    d.q_stride, d.k_stride, d.v_stride = _strides(q), _strides(k), _strides(v)
    d.B, d.Tq, d.Tk, d.Hq, d.Hkv, d.D, d.causal = B, Tq, Tk, Hq, Hkv, D, int(bool(causal))
    d.scale = scale if scale is not None else 1.0 / math.sqrt(D)
    return d, dev, (q, k, v, key_mask)


def _attn_workspace(name, d, grad, dev):
    size = int(L.lib.mic_attn_seq_workspace_bytes(C.byref(d), grad))
    if size < 0:
        L.check(size, name)
    if size == 0:
        return None
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    d.workspace, d.workspace_bytes = ws.data_ptr(), size
    return ws


def attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = False, key_mask: Optional[torch.Tensor] = None,
                      scale: Optional[float] = None):
    """softmax(scale * q k^T) v over whole sequences (models/transformer.py:81-86,130-140): returns ``(o, lse)``.

    q (B, Tq, Hq, D); k, v (B, Tk, Hkv, D), Hq a multiple of Hkv (query head h reads key head h // (Hq // Hkv)); any strides, e.g.
    slices of one packed projection.  ``causal``: query i sees keys up to i + Tk - Tq.  key_mask (B, Tk) bool: True where a key may
    be seen; what k and v hold elsewhere is never used.  A query that sees nothing gets zeros.  scale defaults to D ** -0.5.
    o (B, Tq, Hq, D) in q's dtype, lse (B, Hq, Tq) fp32.  D at most 256 and a multiple of 8 (bf16) or 4 (fp32)."""
    name = "attention_forward"
    d, dev, keep = _attn_desc(name, q, k, v, causal, key_mask, scale)
    o = torch.empty(q.shape, dtype=q.dtype, device=dev)
    lse = torch.empty(q.shape[0], q.shape[2], q.shape[1], dtype=torch.float32, device=dev)
    d.o, d.o_stride, d.lse = o.data_ptr(), _strides(o), lse.data_ptr()
    with torch.cuda.device(dev):
        ws = _attn_workspace(name, d, 0, dev)  # noqa: F841  (alive until the launch is enqueued)
        L.check(L.lib.mic_attn_seq(C.byref(d), _stream(dev)), "mic_attn_seq")
    return o, lse


def attention_grad(grad: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor, *,
                   causal: bool = False, key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None):
    """Gradients ``(dq, dk, dv)`` of ``attention_forward`` for the gradient of o, from its inputs and both results.  The probabilities
    are recomputed; gradients of shared key heads are summed over their query heads in a fixed order."""
    name = "attention_grad"
    d, dev, keep = _attn_desc(name, q, k, v, causal, key_mask, scale)
    _device(name, q, grad, o, lse)
    _need(grad.shape == q.shape and o.shape == q.shape and grad.dtype == q.dtype and o.dtype == q.dtype, name,
          f"grad {tuple(grad.shape)} {grad.dtype} and o {tuple(o.shape)} {o.dtype} do not fit q {tuple(q.shape)} {q.dtype}")
    _need(lse.shape == (q.shape[0], q.shape[2], q.shape[1]) and lse.dtype == torch.float32, name, f"lse {tuple(lse.shape)} {lse.dtype} does not fit q")
    o, grad, lse = _heads(o), _heads(grad), lse.contiguous()
    dq, dk, dv = (torch.empty(t.shape, dtype=q.dtype, device=dev) for t in (q, k, v))
    d.o, d.o_stride, d.lse = o.data_ptr(), _strides(o), lse.data_ptr()
    d.grad_o, d.g_stride = grad.data_ptr(), _strides(grad)
    d.dq, d.dk, d.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    with torch.cuda.device(dev):
        ws = _attn_workspace(name, d, 1, dev)  # noqa: F841
        L.check(L.lib.mic_attn_seq_grad(C.byref(d), _stream(dev)), "mic_attn_seq_grad")
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal, key_mask, scale):
        o, lse = attention_forward(q, k, v, causal=causal, key_mask=key_mask, scale=scale)
        ctx.save_for_backward(q, k, v, o, lse, key_mask)
        ctx.meta = (causal, scale)
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        q, k, v, o, lse, key_mask = ctx.saved_tensors
        causal, scale = ctx.meta
        return (*attention_grad(grad, q, k, v, o, lse, causal=causal, key_mask=key_mask, scale=scale), None, None, None)


def attention(q, k, v, *, causal: bool = False, key_mask=None, scale: Optional[float] = None) -> torch.Tensor:
    """The output of ``attention_forward``, differentiable by ``torch.autograd`` with respect to q, k and v."""
    return _Attention.apply(q, k, v, causal, key_mask, scale)


# ---- vocabulary loss ----------------------------------------------------------------------------------------------------
def _vocab_desc(name, x, w, targets, bias, ignore):
    dev = _device(name, x, w, targets, bias)
    _need(x.dim() == 2 and w.dim() == 2 and x.shape[1] == w.shape[1] and x.shape[1] > 0 and w.shape[0] > 0, name,
          f"x {tuple(x.shape)} and w {tuple(w.shape)} do not fit")
    _need(x.dtype == w.dtype, name, f"x is {x.dtype}, w {w.dtype}")
    N, H = x.shape
    V = w.shape[0]
    _need(targets.shape == (N,), name, f"targets {tuple(targets.shape)} do not fit {N} rows")
    d = L.VocabLossDesc()
    d.dtype = _float_code(name, "x", x.dtype)
    x = x if x.stride(1) == 1 and (N <= 1 or x.stride(0) >= H) else x.contiguous()
    w = w if w.stride(1) == 1 and (V <= 1 or w.stride(0) >= H) else w.contiguous()
    targets = _ids(name, "targets", targets)
    if bias is not None:
        _need(bias.shape == (V,) and bias.dtype == torch.float32, name, f"bias must be float32 ({V},), got {bias.dtype} {tuple(bias.shape)}")
        bias = bias.contiguous()
    ignore = tuple(int(i) for i in ignore)
    _need(len(ignore) <= 4, name, f"{len(ignore)} ignored words (at most 4)")
    d.x, d.w, d.bias, d.targets = x.data_ptr(), w.data_ptr(), L.ptr(bias), targets.data_ptr()
    d.ld_x, d.ld_w = (x.stride(0) if N > 1 else H), (w.stride(0) if V > 1 else H)
    d.N, d.H, d.V, d.target_bits, d.n_ignore = N, H, V, 64 if targets.dtype == torch.int64 else 32, len(ignore)
    for i, v in enumerate(ignore):
        _need(-(1 << 31) <= v < (1 << 31), name, f"ignored word {v}")
        d.ignore[i] = v
    return d, dev, (x, w, targets, bias)


def _vocab_workspace(name, d, grad, dev):
    size = int(L.lib.mic_vocab_loss_workspace_bytes(C.byref(d), grad))
    if size < 0:
        L.check(size, name)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    d.workspace, d.workspace_bytes = ws.data_ptr(), size
    return ws


def vocab_loss_forward(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, *, bias: Optional[torch.Tensor] = None, ignore=()):
    """Cross entropy of every row of x (N, H) against the vocabulary w (V, H) without keeping the logits x w^T + bias (the output
    layer and loss of models/transformer.py:293, train.py:318-354): returns ``(loss, lse)``, both fp32 (N,).

    targets (N,) int32 / int64; rows whose target is in ``ignore`` (at most four words, e.g. padding) or outside the vocabulary
    have loss 0.  bias (V,) fp32."""
    name = "vocab_loss_forward"
    d, dev, keep = _vocab_desc(name, x, w, targets, bias, ignore)
    loss = torch.empty(x.shape[0], dtype=torch.float32, device=dev)
    lse = torch.empty_like(loss)
    d.loss, d.lse = loss.data_ptr(), lse.data_ptr()
    with torch.cuda.device(dev):
        ws = _vocab_workspace(name, d, 0, dev)  # noqa: F841  (alive until the launches are enqueued)
        L.check(L.lib.mic_vocab_loss(C.byref(d), _stream(dev)), "mic_vocab_loss")
    return loss, lse


def vocab_loss_grad(grad: torch.Tensor, x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, lse: torch.Tensor, *,
                    bias: Optional[torch.Tensor] = None, ignore=()):
    """Gradients ``(dx, dw, dbias or None)`` of ``vocab_loss_forward`` for the gradient ``grad`` (N,) fp32 of its losses (a scalar tensor is
    taken for every row), from its inputs and lse.  Rows that do not count get zeros."""
    name = "vocab_loss_grad"
    d, dev, keep = _vocab_desc(name, x, w, targets, bias, ignore)
    _device(name, x, grad, lse)
    N = x.shape[0]
    _need(grad.dtype == torch.float32 and grad.shape in ((N,), ()), name, f"grad must be float32 ({N},), got {grad.dtype} {tuple(grad.shape)}")
    _need(lse.dtype == torch.float32 and lse.shape == (N,), name, f"lse must be float32 ({N},), got {lse.dtype} {tuple(lse.shape)}")
    grad, lse = grad.expand(N).contiguous(), lse.contiguous()
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
    dw = torch.empty(w.shape, dtype=w.dtype, device=dev)
    db = None if bias is None else torch.empty(w.shape[0], dtype=torch.float32, device=dev)
    d.grad_rows, d.lse = grad.data_ptr(), lse.data_ptr()
    d.dx, d.dw, d.db = dx.data_ptr(), dw.data_ptr(), L.ptr(db)
    with torch.cuda.device(dev):
        ws = _vocab_workspace(name, d, 1, dev)  # noqa: F841
        L.check(L.lib.mic_vocab_loss_grad(C.byref(d), _stream(dev)), "mic_vocab_loss_grad")
    return dx, dw, db


class _VocabLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, targets, bias, ignore):
        loss, lse = vocab_loss_forward(x, w, targets, bias=bias, ignore=ignore)
        ctx.save_for_backward(x, w, targets, bias, lse)
        ctx.ignore = ignore
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, w, targets, bias, lse = ctx.saved_tensors
        dx, dw, db = vocab_loss_grad(grad, x, w, targets, lse, bias=bias, ignore=ctx.ignore)
        return dx, dw, None, db, None


def vocab_loss(x, w, targets, *, bias=None, ignore=()) -> torch.Tensor:
    """The losses (N,) of ``vocab_loss_forward``, differentiable by ``torch.autograd`` with respect to x, w and bias; sum, average or
    weight them as the training step wants (train.py:346-352 averages over the counted rows)."""
    return _VocabLoss.apply(x, w, targets, bias, tuple(ignore))
