"""8-bit floating point (e4m3) with a scale for each block of 128: quantising, and the lm_head product on it.

`quantize_fp8` turns activations (a scale per 1 x 128 elements) or a weight (per 128 x 128) into `Fp8Blocks`;
`fp8_matmul` multiplies the two, `x @ w.T`, on the tensor cores, each block's inner sum and the sum over blocks in
f32.  `linear_loss.lm_head_forward` takes a head quantised this way in place of a bf16 weight: the log-probs of a
frozen reference model from half the memory.  Nothing here is differentiable: it is the form in which a model is
read, not trained.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib

BLOCK = 128
_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}


class Fp8Blocks:
    """values e4m3 [R, C] and scales f32 [ceil(R / block[0]), ceil(C / 128)]; the tensor they stand for is
    values * scale of the block.  block is (1, 128) or (128, 128)."""

    __slots__ = ("values", "scales", "block")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor, block: Tuple[int, int] = (128, 128)):
        if tuple(block) not in ((1, BLOCK), (BLOCK, BLOCK)):
            raise ValueError(f"block must be (1, 128) or (128, 128), got {block}")
        if values.dtype != torch.float8_e4m3fn or values.dim() != 2:
            raise TypeError(f"values must be float8_e4m3fn [R, C], got {values.dtype} {tuple(values.shape)}")
        R, C = values.shape
        want = (-(-R // block[0]), -(-C // BLOCK))
        if scales.dtype != torch.float32 or tuple(scales.shape) != want or scales.device != values.device:
            raise ValueError(f"scales must be float32 {want} on the values' device, got {scales.dtype} {tuple(scales.shape)}")
        if not scales.is_contiguous():
            scales = scales.contiguous()
        self.values, self.scales, self.block = values, scales, tuple(block)

    @property
    def shape(self):
        return self.values.shape

    @property
    def device(self):
        return self.values.device

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The tensor the blocks stand for (torch operations; a check, not a hot path)."""
        R, C = self.values.shape
        s = self.scales.repeat_interleave(BLOCK, 1)[:, :C]
        if self.block[0] != 1:
            s = s.repeat_interleave(BLOCK, 0)[:R]
        return (self.values.to(torch.float32) * s).to(dtype)


def quantize_fp8(x: torch.Tensor, *, block: Tuple[int, int] = (1, BLOCK)) -> Fp8Blocks:
    """x [R, C] bf16 / f16 / f32 (rows any distance apart) -> Fp8Blocks with q = e4m3(448 x / amax of the block), to
    nearest even, and scale = amax / 448 (at least 2^-126).  Blocks at the edges are shorter.  16-bit inputs are rounded
    exactly so; of f32 inputs a quotient within 2^-19 (relative) of the middle between two values counts as the middle."""
    if not x.is_cuda:
        raise RuntimeError("quantize_fp8 needs CUDA tensors: the kernels have no CPU path")
    if x.dtype not in _DTYPES:
        raise TypeError(f"x must be bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"x must be [R, C], got shape {tuple(x.shape)}")
    if tuple(block) not in ((1, BLOCK), (BLOCK, BLOCK)):
        raise ValueError(f"block must be (1, 128) or (128, 128), got {block}")
    R, C = x.shape
    if (x.stride(1) != 1 and C > 1) or (R > 1 and x.stride(0) < C):
        x = x.contiguous()
    dev = x.device
    values = torch.empty(R, C, dtype=torch.float8_e4m3fn, device=dev)
    scales = torch.empty(-(-R // block[0]), -(-C // BLOCK), dtype=torch.float32, device=dev)
    a = _lib.Fp8QuantizeArgs()
    a.rows, a.cols, a.x_stride, a.q_stride = R, C, max(x.stride(0), C), C
    a.block_rows, a.dtype = block[0], _DTYPES[x.dtype]
    a.x, a.q, a.scales = x.data_ptr(), values.data_ptr(), scales.data_ptr()
    _lib.launch("mllm_lm_head_fp8_quantize", a, dev)
    return Fp8Blocks(values, scales, block)


def _operand(t: Fp8Blocks, name: str, block) -> Tuple[int, int, int, int]:
    """Rows, columns, bytes between rows and address of the values, as the tensor-core kernels read them: 16-byte rows
    at 16-byte addresses."""
    if t.block != block:
        raise ValueError(f"{name} must have blocks of {block}, got {t.block}")
    R, C = t.values.shape
    row, col = t.values.stride()
    at = t.values.data_ptr()
    if C % 16:
        raise ValueError(f"the inner size must be a multiple of 16, got {C}")
    if R == 1:
        row = C
    if col != 1 or row < C or row % 16 or at % 16:
        raise ValueError(f"{name} needs contiguous rows that start on 16-byte boundaries")
    return R, C, row, at


def _bind(x: Fp8Blocks, w: Fp8Blocks) -> _lib.Fp8Args:
    M, K, x_stride, x_at = _operand(x, "x", (1, BLOCK))
    N, w_inner, w_stride, w_at = _operand(w, "w", (BLOCK, BLOCK))
    if not x.values.is_cuda:
        raise RuntimeError("the 8-bit product needs CUDA tensors: the kernels have no CPU path")
    if K != w_inner or x.device != w.device or N < 1:
        raise ValueError(f"x {tuple(x.shape)} on {x.device} and w {tuple(w.shape)} on {w.device} do not match")
    return _lib.Fp8Args(n_rows=M, vocab=N, hidden_dim=K, hidden_stride=x_stride, weight_stride=w_stride, hidden=x_at,
                        hidden_scales=x.scales.data_ptr(), weight=w_at, weight_scales=w.scales.data_ptr())


def _quantize_and_bind(x: torch.Tensor, w: Fp8Blocks, room: int) -> Tuple[_lib.Fp8Args, torch.Tensor, int]:
    """Rows x [M, K] quantised into one buffer and bound with w; the buffer has `room` more bytes from the returned place
    on (16-byte aligned).  One allocation: a small call is bound by the host."""
    N, K, w_stride, w_at = _operand(w, "w", (BLOCK, BLOCK))
    M, dev = x.shape[0], x.device
    if dev != w.device or x.shape[1] != K or N < 1:
        raise ValueError(f"x {tuple(x.shape)} on {dev} and w {tuple(w.shape)} on {w.device} do not match")
    if x.stride(1) != 1 or (M > 1 and x.stride(0) < K):
        x = x.contiguous()
    scales = M * K
    end = scales + (4 * M * -(-K // BLOCK) + 15) // 16 * 16
    buf = torch.empty(end + room, dtype=torch.uint8, device=dev)
    at = buf.data_ptr()
    _lib.launch("mllm_lm_head_fp8_quantize", _lib.Fp8QuantizeArgs(
        rows=M, cols=K, x_stride=x.stride(0) if M > 1 else K, q_stride=K, block_rows=1, dtype=_DTYPES[x.dtype],
        x=x.data_ptr(), q=at, scales=at + scales), dev)
    return _lib.Fp8Args(n_rows=M, vocab=N, hidden_dim=K, hidden_stride=K, weight_stride=w_stride, hidden=at,
                        hidden_scales=at + scales, weight=w_at, weight_scales=w.scales.data_ptr()), buf, end


def fp8_matmul(x: Union[Fp8Blocks, torch.Tensor], w: Fp8Blocks, *, out_dtype: torch.dtype = torch.bfloat16,
               out: Optional[torch.Tensor] = None, device_status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [M, K] (Fp8Blocks with blocks of (1, 128), or a tensor, which is quantised first) times w [N, K] (blocks of
    (128, 128)), transposed: [M, N] of out_dtype (bf16, f16 or f32), rounded once.  K must be a multiple of 16.
    `out` [M, N] (rows any distance apart) is written instead of a new tensor when given.  If a wait inside the kernel runs
    out, the elements that were not reached are NaN and device_status (an int32 CUDA tensor of the caller), where one is
    passed, has MLLM_GRPO_DEV_WAIT_TIMEOUT set."""
    if not isinstance(x, Fp8Blocks):
        x = quantize_fp8(x, block=(1, BLOCK))
    a = _bind(x, w)
    M, N = x.shape[0], w.shape[0]
    given = out is not None
    if not given:
        if out_dtype not in _DTYPES:
            raise TypeError(f"out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
        out = torch.empty(M, N, dtype=out_dtype, device=x.device)
    elif tuple(out.shape) != (M, N) or out.dtype not in _DTYPES or out.device != x.device or \
            (out.stride(1) != 1 and N > 1) or (M > 1 and out.stride(0) < N):
        raise ValueError(f"out must be [{M}, {N}] of bfloat16, float16 or float32 on {x.device} with contiguous rows")
    a.out_stride, a.out_dtype, a.out = max(out.stride(0), N) if M > 1 else N, _DTYPES[out.dtype], out.data_ptr()
    if device_status is not None:
        a.device_status = _lib.status_word(device_status, x.device)
    _lib.launch("mllm_lm_head_fp8_matmul", a, x.device)
    if given:
        _lib.written(out)
    return out
