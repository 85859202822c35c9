"""Teacher-forced operators of the caption decoders on whole sequences, with their gradients.

The decode path takes one position at a time and needs no gradient; a training or scoring step (train.py:163-262 of the
reference) takes whole captions.  Each operator comes as a pair of plain calls, ``*_forward`` and ``*_grad``, that enqueue
kernels on the current stream of the tensors' device and return new tensors, and as one differentiable call for
``torch.autograd`` built on the pair: ``embedding``, ``attention``, ``vocab_loss``.

Tensors live on one HIP device, fp32 or bf16.  Nothing synchronises; every call may be captured into a HIP graph (workspaces
come from torch's allocator, which gives a captured graph a pool of its own).  Capture the plain calls, or ``torch.autograd.grad``
of the differentiable ones: a captured ``.backward()`` into leaves that an eager graph still holds ends the process inside torch.
Refused arguments raise ``ValueError`` (shapes, types, devices) or ``_lib.MicError`` (what the library refuses).
"""
from __future__ import annotations

import functools
import math
import struct
from typing import Optional

import torch

from . import _lib as L

_raw_stream = torch._C._cuda_getCurrentRawStream  # what torch.cuda.current_stream(i).cuda_stream returns, without building the object

__all__ = ["embedding", "embedding_forward", "embedding_grad", "attention", "attention_forward", "attention_grad",
           "vocab_loss", "vocab_loss_forward", "vocab_loss_grad"]


# These calls are a few microseconds of host work around launches that can be as short, so the checks build their messages only
# when they fail, and the descriptors are packed in one go instead of field by field.
def _device(name: str, *tensors) -> int:
    """Ordinal of the one HIP device all given tensors (None is skipped) live on."""
    dev = -1
    for t in tensors:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{name}: expected tensors, got {type(t).__name__}")
        if not t.is_cuda:
            raise ValueError(f"{name}: tensors must be on a HIP device, got one on {t.device}")
        i = t.get_device()
        if dev != i and dev >= 0:
            raise ValueError(f"{name}: tensors are on devices {dev} and {i}")
        dev = i
    return dev


def _float_code(name: str, what: str, dtype) -> int:
    if dtype is torch.float32:
        return L.F32
    if dtype is torch.bfloat16:
        return L.BF16
    raise ValueError(f"{name}: {what} must be float32 or bfloat16, got {dtype}")


def _workspace(size: int, like: torch.Tensor):
    """`size` bytes of scratch and its address; the caller keeps the tensor until its launches are enqueued."""
    if size == 0:
        return None, 0
    ws = torch.empty(size, dtype=torch.uint8, device=like.device)
    return ws, ws.data_ptr()


def _ids(name: str, what: str, t: torch.Tensor) -> torch.Tensor:
    if t.dtype is not torch.int64 and t.dtype is not torch.int32:
        raise ValueError(f"{name}: {what} must be int32 or int64, got {t.dtype}")
    return t.contiguous()


def _small(name: str, *sizes) -> None:
    """The library takes sizes of 32 bits."""
    if max(sizes) >= 1 << 31:
        raise ValueError(f"{name}: sizes out of range {sizes}")


def _bits(t: torch.Tensor) -> int:
    return 64 if t.dtype is torch.int64 else 32


def _run(what: str, fn, dev: int, *args) -> None:
    """fn(*args, current stream of the device), with that device current."""
    if torch.cuda.current_device() == dev:
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc != 0:
        L.check(rc, what)


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A matrix whose rows are consecutive in memory and do not overlap (the tensor itself where it is one)."""
    if t.stride(1) == 1 and (t.stride(0) >= t.shape[1] or t.shape[0] == 1):
        return t
    return t.contiguous()


# ---- embedding --------------------------------------------------------------------------------------------------------
def embedding_forward(ids: torch.Tensor, table: torch.Tensor, pos: Optional[torch.Tensor] = None, *, scale: float = 1.0,
                      dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``scale * table[ids] + pos`` rounded once to ``dtype`` (the table's by default); models/transformer.py:44-50.

    ids (..., T) int32 / int64; table (vocab, H); pos (at least T rows, H) in the table's dtype, row t added at position t of the
    last dimension of ids.  Ids outside the vocabulary read its nearest row.  Returns (..., T, H)."""
    name = "embedding_forward"
    dev = _device(name, ids, table, pos)
    if table.dim() != 2 or table.numel() == 0:
        raise ValueError(f"{name}: table must be (vocab, H), got {tuple(table.shape)}")
    if ids.dim() < 1:
        raise ValueError(f"{name}: ids need at least one dimension")
    vocab, H = table.shape
    T = ids.shape[-1]
    _small(name, vocab, H, T)
    code = _float_code(name, "the table", table.dtype)
    out_dtype = table.dtype if dtype is None else dtype
    out_code = _float_code(name, "the output", out_dtype)
    pos_ptr, ld_pos = None, 0
    if pos is not None:
        if pos.dim() != 2 or pos.shape[1] != H or pos.shape[0] < T or pos.dtype is not table.dtype:
            raise ValueError(f"{name}: pos must be (>= {T}, {H}) of {table.dtype}, got {tuple(pos.shape)} of {pos.dtype}")
        pos = _rows(pos)
        pos_ptr, ld_pos = pos.data_ptr(), max(pos.stride(0), H)
    table = _rows(table)
    ids = _ids(name, "ids", ids)
    out = torch.empty((*ids.shape, H), dtype=out_dtype, device=table.device)
    n = ids.numel()
    if n:
        _run("mic_embed_rows", L.lib.mic_embed_rows, dev, ids.data_ptr(), _bits(ids), table.data_ptr(), max(table.stride(0), H), pos_ptr, ld_pos,
             out.data_ptr(), code, out_code, scale, n, T, H, vocab)
    return out


@functools.lru_cache(maxsize=256)
def _embed_workspace_bytes(n, T, H, vocab, want_pos) -> int:
    return L.lib.mic_embed_grad_workspace_bytes(n, T, H, vocab, want_pos)


def embedding_grad(grad: torch.Tensor, ids: torch.Tensor, vocab: int, *, scale: float = 1.0, positions: int = 0,
                   dtype: Optional[torch.dtype] = None):
    """Gradients of ``embedding_forward``: (d_table (vocab, H), d_pos (positions, H) or None), rounded once to ``dtype`` (grad's by
    default).  grad (..., T, H) is the gradient of the output; positions is the row count of the positional table, 0 for none.
    Sums run in fp32 over the tokens sorted by word: the same inputs give the same bits."""
    name = "embedding_grad"
    dev = _device(name, grad, ids)
    if ids.dim() < 1 or grad.shape[:-1] != ids.shape:
        raise ValueError(f"{name}: grad {tuple(grad.shape)} does not fit ids {tuple(ids.shape)}")
    H, T, n = grad.shape[-1], ids.shape[-1], ids.numel()
    if H < 1 or vocab < 1:
        raise ValueError(f"{name}: bad sizes H={H} vocab={vocab}")
    _small(name, vocab, H, T, positions)
    if positions and positions < T:
        raise ValueError(f"{name}: {positions} positions for sequences of {T}")
    code = _float_code(name, "grad", grad.dtype)
    out_dtype = grad.dtype if dtype is None else dtype
    out_code = _float_code(name, "the gradients", out_dtype)
    ids, grad = _ids(name, "ids", ids), grad.contiguous()
    d_table = torch.empty((vocab, H), dtype=out_dtype, device=grad.device)
    d_pos = None
    if positions:
        d_pos = torch.empty((positions, H), dtype=out_dtype, device=grad.device)
        if positions > T:
            d_pos[T:].zero_()
    T = max(T, 1)
    size = _embed_workspace_bytes(n, T, H, vocab, 1 if positions else 0)
    if size < 0:
        raise ValueError(f"{name}: sizes out of range (tokens {n}, H={H}, vocab={vocab})")
    ws, ws_ptr = _workspace(size, grad)
    _run("mic_embed_grad", L.lib.mic_embed_grad, dev, ids.data_ptr(), _bits(ids), grad.data_ptr(), d_table.data_ptr(), L.ptr(d_pos), code, out_code,
         scale, n, T, H, vocab, ws_ptr, size)
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
_ATTN_PACK = struct.Struct("@10P16q8ifPq")  # mic_attn_seq_desc

@functools.lru_cache(maxsize=256)
def _attn_workspace_bytes(code, B, Tq, Tk, Hq, Hkv, D, causal, grad) -> int:
    """Scratch depends on type, sizes and causality alone."""
    d = L.AttnSeqDesc.from_buffer_copy(_ATTN_PACK.pack(*(0,) * 26, code, B, Tq, Tk, Hq, Hkv, D, causal, 0.0, 0, 0))
    size = L.lib.mic_attn_seq_workspace_bytes(d, grad)
    if size < 0:
        L.check(size, "mic_attn_seq_workspace_bytes")
    return size


def _heads(t: torch.Tensor):
    """The tensor, its address and its strides of (batch, position, head), copied if the kernels cannot read it in place (columns
    consecutive, everything on 16-byte boundaries, 64 positions and the heads of one within 1 GiB).  A dimension of one entry has no
    stride to speak of."""
    e = 16 // t.element_size()
    B, T, H, D = t.shape
    p = t.data_ptr()
    sb, st, sh, sd = t.stride()
    if B == 1:
        sb = 0
    if T == 1:
        st = 0
    if H == 1:
        sh = 0
    if not (sb % e or st % e or sh % e or p % 16) and (sd == 1 or D == 1) and st <= e << 20 and sh * H <= e << 26:
        return t, p, (sb, st, sh)
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.data_ptr(), (T * H * D, H * D, D)


def _attn_check(name, dev, q, k, v, key_mask):
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError(f"{name}: q, k and v must be (batch, positions, heads, columns), got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, Tq, Hq, D = q.shape
    Bk, Tk, Hkv, Dk = k.shape
    if Bk != B or Dk != D or Hq < 1 or Hkv < 1 or D < 1:
        raise ValueError(f"{name}: q {tuple(q.shape)} and k {tuple(k.shape)} do not fit")
    _small(name, B, Tq, Tk, Hq, Hkv, D)
    dtype = q.dtype
    if k.dtype is not dtype or v.dtype is not dtype:
        raise ValueError(f"{name}: q, k and v are {dtype}, {k.dtype} and {v.dtype}")
    code = _float_code(name, "q", dtype)
    mask_ptr, mask_stride = 0, 0
    if key_mask is not None:
        if key_mask.dtype not in (torch.bool, torch.uint8) or key_mask.shape != (B, Tk):
            raise ValueError(f"{name}: key_mask must be bool ({B}, {Tk}), got {key_mask.dtype} {tuple(key_mask.shape)}")
        if Tk > 1 and key_mask.stride(1) != 1:
            key_mask = key_mask.contiguous()
        mask_ptr, mask_stride = key_mask.data_ptr(), key_mask.stride(0)
    return code, B, Tq, Tk, Hq, Hkv, D, dtype, key_mask, mask_ptr, mask_stride


def attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = False, key_mask: Optional[torch.Tensor] = None,
                      scale: Optional[float] = None):
    """softmax(scale * q k^T) v over whole sequences (models/transformer.py:81-86,130-140): returns ``(o, lse)``.

    q (B, Tq, Hq, D); k, v (B, Tk, Hkv, D), Hq a multiple of Hkv (query head h reads key head h // (Hq // Hkv)); any strides, e.g.
    slices of one packed projection.  ``causal``: query i sees keys up to i + Tk - Tq.  key_mask (B, Tk) bool: True where a key may
    be seen; what k and v hold elsewhere is never used.  (A key hidden from a query by causality alone takes part in its products with
    weight zero, so it has to be finite.)  A query that sees nothing gets zeros, whatever it holds.  scale defaults to D ** -0.5.
    o (B, Tq, Hq, D) in q's dtype, lse (B, Hq, Tq) fp32.  D at most 256 and a multiple of 8 (bf16) or 4 (fp32)."""
    name = "attention_forward"
    dev = _device(name, q, k, v, key_mask)
    code, B, Tq, Tk, Hq, Hkv, D, dtype, key_mask, mask_ptr, mask_stride = _attn_check(name, dev, q, k, v, key_mask)
    q, q_ptr, qs = _heads(q)
    k, k_ptr, ks = _heads(k)
    v, v_ptr, vs = _heads(v)
    place = q.device
    o = torch.empty((B, Tq, Hq, D), dtype=dtype, device=place)
    lse = torch.empty((B, Hq, Tq), dtype=torch.float32, device=place)
    causal = 1 if causal else 0
    size = _attn_workspace_bytes(code, B, Tq, Tk, Hq, Hkv, D, causal, 0)
    ws, ws_ptr = _workspace(size, q)
    _run("mic_attn_seq", L.lib.mic_attn_seq, dev, L.AttnSeqDesc.from_buffer_copy(_ATTN_PACK.pack(
        q_ptr, k_ptr, v_ptr, o.data_ptr(), lse.data_ptr(), mask_ptr, 0, 0, 0, 0, *qs, *ks, *vs, Tq * Hq * D, Hq * D, D, 0, 0, 0, mask_stride, code, B, Tq,
        Tk, Hq, Hkv, D, causal, 1.0 / math.sqrt(D) if scale is None else scale, ws_ptr, size)))
    return o, lse


def attention_grad(grad: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor, *,
                   causal: bool = False, key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None):
    """Gradients ``(dq, dk, dv)`` of ``attention_forward`` for the gradient of o, from its inputs and both results.  The probabilities
    are recomputed; gradients of shared key heads are summed over their query heads in a fixed order."""
    name = "attention_grad"
    dev = _device(name, q, k, v, key_mask, grad, o, lse)
    code, B, Tq, Tk, Hq, Hkv, D, dtype, key_mask, mask_ptr, mask_stride = _attn_check(name, dev, q, k, v, key_mask)
    if grad.shape != q.shape or o.shape != q.shape or grad.dtype is not dtype or o.dtype is not dtype:
        raise ValueError(f"{name}: grad {tuple(grad.shape)} {grad.dtype} and o {tuple(o.shape)} {o.dtype} do not fit q {tuple(q.shape)} {dtype}")
    if lse.shape != (B, Hq, Tq) or lse.dtype is not torch.float32:
        raise ValueError(f"{name}: lse {tuple(lse.shape)} {lse.dtype} does not fit q {tuple(q.shape)}")
    q, q_ptr, qs = _heads(q)
    k, k_ptr, ks = _heads(k)
    v, v_ptr, vs = _heads(v)
    o, o_ptr, os = _heads(o)
    grad, g_ptr, gs = _heads(grad)
    lse = lse.contiguous()
    place = q.device
    dq = torch.empty((B, Tq, Hq, D), dtype=dtype, device=place)
    dk = torch.empty((B, Tk, Hkv, D), dtype=dtype, device=place)
    dv = torch.empty((B, Tk, Hkv, D), dtype=dtype, device=place)
    causal = 1 if causal else 0
    size = _attn_workspace_bytes(code, B, Tq, Tk, Hq, Hkv, D, causal, 1)
    ws, ws_ptr = _workspace(size, q)
    _run("mic_attn_seq_grad", L.lib.mic_attn_seq_grad, dev, L.AttnSeqDesc.from_buffer_copy(_ATTN_PACK.pack(
        q_ptr, k_ptr, v_ptr, o_ptr, lse.data_ptr(), mask_ptr, g_ptr, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), *qs, *ks, *vs, *os, *gs, mask_stride,
        code, B, Tq, Tk, Hq, Hkv, D, causal, 1.0 / math.sqrt(D) if scale is None else scale, ws_ptr, size)))
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
_VOCAB_PACK = struct.Struct("@10P2q6i4iPq")  # mic_vocab_loss_desc


def _vocab_check(name, x, w, targets, bias, ignore):
    dev = _device(name, x, w, targets, bias)
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1] or w.numel() == 0:
        raise ValueError(f"{name}: x {tuple(x.shape)} and w {tuple(w.shape)} do not fit")
    if x.dtype is not w.dtype:
        raise ValueError(f"{name}: x is {x.dtype}, w {w.dtype}")
    N, H = x.shape
    V = w.shape[0]
    _small(name, N, H, V)
    if targets.shape != (N,):
        raise ValueError(f"{name}: targets {tuple(targets.shape)} do not fit {N} rows")
    code = _float_code(name, "x", x.dtype)
    if bias is not None:
        if bias.shape != (V,) or bias.dtype is not torch.float32:
            raise ValueError(f"{name}: bias must be float32 ({V},), got {bias.dtype} {tuple(bias.shape)}")
        bias = bias.contiguous()
    ignore = tuple(ignore)
    if len(ignore) > 4 or any(not -(1 << 31) <= i < (1 << 31) for i in ignore):
        raise ValueError(f"{name}: at most four ignored words of 32 bits, got {ignore}")
    return dev, code, N, H, V, _rows(x), _rows(w), _ids(name, "targets", targets), bias, ignore


def _vocab_call(what, fn, grad, dev, code, N, H, V, x, w, targets, bias, ignore, loss, lse, grad_rows, dx, dw, db):
    d = L.VocabLossDesc.from_buffer_copy(_VOCAB_PACK.pack(
        x.data_ptr(), w.data_ptr(), _ptr(bias), targets.data_ptr(), _ptr(loss), lse.data_ptr(), _ptr(grad_rows), _ptr(dx), _ptr(dw), _ptr(db),
        max(x.stride(0), H), max(w.stride(0), H), code, N, H, V, _bits(targets), len(ignore), *ignore, *(0,) * (4 - len(ignore)), 0, 0))
    size = L.lib.mic_vocab_loss_workspace_bytes(d, grad)
    if size < 0:
        L.check(size, what)
    ws, ws_ptr = _workspace(size, x)
    if size:
        d.workspace, d.workspace_bytes = ws_ptr, size
    _run(what, fn, dev, d)


def vocab_loss_forward(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, *, bias: Optional[torch.Tensor] = None, ignore=()):
    """Cross entropy of every row of x (N, H) against the vocabulary w (V, H) without keeping the logits x w^T + bias (the output
    layer and loss of models/transformer.py:293, train.py:318-354): returns ``(loss, lse)``, both fp32 (N,).

    targets (N,) int32 / int64; rows whose target is in ``ignore`` (at most four words, e.g. padding) or outside the vocabulary
    have loss 0.  bias (V,) fp32."""
    dev, code, N, H, V, x, w, targets, bias, ignore = _vocab_check("vocab_loss_forward", x, w, targets, bias, ignore)
    loss = torch.empty(N, dtype=torch.float32, device=x.device)
    lse = torch.empty(N, dtype=torch.float32, device=x.device)
    _vocab_call("mic_vocab_loss", L.lib.mic_vocab_loss, 0, dev, code, N, H, V, x, w, targets, bias, ignore, loss, lse, None, None, None, None)
    return loss, lse


def vocab_loss_grad(grad: torch.Tensor, x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, lse: torch.Tensor, *,
                    bias: Optional[torch.Tensor] = None, ignore=()):
    """Gradients ``(dx, dw, dbias or None)`` of ``vocab_loss_forward`` for the gradient ``grad`` (N,) fp32 of its losses (a scalar tensor is
    taken for every row), from its inputs and lse.  Rows that do not count get zeros."""
    name = "vocab_loss_grad"
    dev, code, N, H, V, x, w, targets, bias, ignore = _vocab_check(name, x, w, targets, bias, ignore)
    _device(name, x, grad, lse)
    if grad.dtype is not torch.float32 or (grad.shape != (N,) and grad.dim() != 0):
        raise ValueError(f"{name}: grad must be float32 ({N},), got {grad.dtype} {tuple(grad.shape)}")
    if lse.dtype is not torch.float32 or lse.shape != (N,):
        raise ValueError(f"{name}: lse must be float32 ({N},), got {lse.dtype} {tuple(lse.shape)}")
    grad, lse = grad.expand(N).contiguous(), lse.contiguous()
    dx = torch.empty((N, H), dtype=x.dtype, device=x.device)
    dw = torch.empty((V, H), dtype=x.dtype, device=x.device)
    db = None if bias is None else torch.empty(V, dtype=torch.float32, device=x.device)
    _vocab_call("mic_vocab_loss_grad", L.lib.mic_vocab_loss_grad, 1, dev, code, N, H, V, x, w, targets, bias, ignore, None, lse, grad, dx, dw, db)
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
