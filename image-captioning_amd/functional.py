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

from typing import Optional

import torch

from . import _lib as L

__all__ = ["embedding", "embedding_forward", "embedding_grad"]


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
