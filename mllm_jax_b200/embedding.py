"""Embedding table at the other end of a tied lm_head: scaled lookup and its gradient by sorted tokens.

    out[n, :] = scale * weight[ids[n], :]           dweight[v, :] = scale * sum_{n: ids[n] = v} grad_out[n, :]

The products are f32, rounded once to the table's type; the gradient's sums are f32 in an order that depends on the
ids alone (a stable sort, no floating-point atomics), so equal calls give equal bits.  `embedding_grad` either writes
a whole new gradient or adds to the f32 `dweight` that `linear_grpo_value_and_grad` returns for a tied head.  A table
that is split over ranks by vocabulary rows passes `vocab_start` and `vocab_total`: ids of other shards give zero rows
(the ranks' outputs add up) and no gradient.  Ids outside [0, vocab_total) give a zero row and no gradient and raise
MLLM_GRPO_DEV_ID_IGNORED in `device_status` (an int32 CUDA tensor of the caller), when one is passed.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}


def _dtype(t: torch.Tensor, name: str) -> int:
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    return _DTYPES[t.dtype]


def _ids(ids: torch.Tensor, dev) -> torch.Tensor:
    if ids.dtype == torch.int64:
        ids = ids.clamp(-1, 2 ** 31 - 1)  # an id beyond 32 bits must not wrap to a valid one
    elif ids.dtype != torch.int32:
        raise TypeError(f"ids must be int32 or int64, got {ids.dtype}")
    return ids.to(device=dev, dtype=torch.int32).contiguous()


def _rows(t: torch.Tensor, hidden: int) -> torch.Tensor:
    """[..., H] as rows evenly spaced (a view where the strides allow it)."""
    t = t.reshape(-1, hidden)
    return t if t.shape[0] == 0 or (t.stride(1) == 1 or hidden == 1) and t.stride(0) >= hidden else t.contiguous()


def _args(n, vocab, hidden, scale, vocab_start, vocab_total, device_status, dev) -> _lib.EmbeddingArgs:
    a = _lib.EmbeddingArgs()
    a.n_tokens, a.vocab, a.hidden = n, vocab, hidden
    a.vocab_start, a.vocab_total = int(vocab_start), 0 if vocab_total is None else int(vocab_total)
    a.scale = float(scale)
    if device_status is not None:
        a.device_status = _lib.status_word(device_status, dev)
    return a


def _lookup(ids, weight, scale, vocab_start, vocab_total, device_status) -> torch.Tensor:
    dev = weight.device
    V, H = weight.shape
    ids32 = _ids(ids, dev)
    out = torch.empty(*ids.shape, H, dtype=weight.dtype, device=dev)
    a = _args(ids32.numel(), V, H, scale, vocab_start, vocab_total, device_status, dev)
    a.weight_stride, a.token_stride = max(weight.stride(0), H), H
    a.dtype = _dtype(weight, "weight")
    a.ids, a.weight, a.out = ids32.data_ptr(), weight.data_ptr(), out.data_ptr()
    _lib.launch("mllm_grpo_embedding_lookup", a, dev)
    return out


class _EmbeddingLookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale, vocab_start, vocab_total, device_status):
        ctx.save_for_backward(ids)
        ctx.shape, ctx.dtype = weight.shape, weight.dtype
        ctx.rest = (scale, vocab_start, vocab_total)
        return _lookup(ids, weight, scale, vocab_start, vocab_total, device_status)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        (ids,) = ctx.saved_tensors
        scale, vocab_start, vocab_total = ctx.rest
        g = embedding_grad(grad_out, ids, ctx.shape[0], scale=scale, vocab_start=vocab_start, vocab_total=vocab_total,
                           dtype=ctx.dtype)
        return g, None, None, None, None, None


def embedding_lookup(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, vocab_start: int = 0,
                     vocab_total: Optional[int] = None, device_status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """ids [...] int32 / int64, weight [V, H] bf16 / f16 / f32 (rows any distance apart) -> [..., H] in weight's type.

    Differentiable with respect to weight: its gradient is `embedding_grad` in weight's type, all [V, H] of it.  Reverse
    mode only: a weight with a forward-mode tangent is refused."""
    if not weight.is_cuda:
        raise RuntimeError("embedding_lookup needs CUDA tensors: the kernels have no CPU path")
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight must be [V, H], got shape {tuple(weight.shape)}")
    if (weight.stride(1) != 1 and weight.shape[1] > 1) or (weight.shape[0] > 1 and weight.stride(0) < weight.shape[1]):
        raise ValueError("weight rows must be contiguous and must not overlap")
    _lib.no_tangent(weight, "weight")
    if weight.requires_grad and torch.is_grad_enabled():
        return _EmbeddingLookup.apply(weight, ids, float(scale), vocab_start, vocab_total, device_status)
    return _lookup(ids, weight, scale, vocab_start, vocab_total, device_status)


def embedding_grad(grad_out: torch.Tensor, ids: torch.Tensor, vocab: int, *, scale: float = 1.0,
                   vocab_start: int = 0, vocab_total: Optional[int] = None, dtype: torch.dtype = torch.float32,
                   out: Optional[torch.Tensor] = None, device_status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of `embedding_lookup` with respect to the table.

    grad_out [..., H] bf16 / f16 / f32, ids [...] -> a new [vocab, H] tensor of `dtype`, every row written.  With
    `out` (f32 [vocab, H], rows any distance apart) the sums are ADDED to it instead and rows without tokens are not
    touched: pass the `dweight` of `linear_grpo_value_and_grad` for a tied table."""
    if not grad_out.is_cuda:
        raise RuntimeError("embedding_grad needs CUDA tensors: the kernels have no CPU path")
    dev = grad_out.device
    if grad_out.dim() < 1 or grad_out.shape[:-1] != ids.shape or grad_out.shape[-1] < 1:
        raise ValueError(f"grad_out {tuple(grad_out.shape)} must be ids {tuple(ids.shape)} with one more dimension")
    _lib.no_tangent(grad_out, "grad_out")
    vocab = int(vocab)
    H = grad_out.shape[-1]
    g = _rows(grad_out, H)
    ids32 = _ids(ids, dev)
    a = _args(ids32.numel(), vocab, H, scale, vocab_start, vocab_total, device_status, dev)
    a.dtype = _dtype(grad_out, "grad_out")
    a.token_stride = max(g.stride(0), H) if g.shape[0] > 1 else H
    if out is None:
        if dtype not in _DTYPES:
            raise TypeError(f"dtype must be bfloat16, float16 or float32, got {dtype}")
        res = torch.empty(vocab, H, dtype=dtype, device=dev)
        a.weight_stride, a.out_dtype = H, _DTYPES[dtype]
    else:
        if tuple(out.shape) != (vocab, H) or out.dtype != torch.float32 or out.device != dev or \
                (out.stride(1) != 1 and H > 1) or (vocab > 1 and out.stride(0) < H):
            raise ValueError(f"out must be float32 [{vocab}, {H}] on {dev} with contiguous rows that do not overlap")
        res = out
        a.weight_stride, a.out_dtype, a.accumulate = max(out.stride(0), H), _lib.DTYPE_F32, 1
    lib = _lib.load()
    nbytes = int(lib.mllm_grpo_embedding_workspace_bytes(a.n_tokens, H, vocab))
    if nbytes == 0:
        raise ValueError(f"{a.n_tokens} tokens, {vocab} rows of {H}: not a size that one call takes")
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    a.ids, a.grad_out, a.dweight, a.workspace = ids32.data_ptr(), g.data_ptr(), res.data_ptr(), workspace.data_ptr()
    _lib.launch("mllm_grpo_embedding_grad", a, dev)
    if out is not None:
        _lib.written(out)
    return res
