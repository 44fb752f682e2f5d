"""Linear layers in 8-bit integers (no counterpart in the reference, whose projections stay fp16).

  quantize_per_token_int8  rows of x -> int8 codes and one fp32 scale a row (activations by token,
                           weights by output channel: the same operation)
  int8_matmul              (x8 . w8^T) * x_scale * w_scale + bias on the tensor cores
  int8_linear              both: what a layer calls
  Int8Linear               an ``nn.Linear`` whose weight is held in 8 bits

``scale = amax / 127``, ``code = 127 x / amax`` rounded half away from zero (the rounding of the
per-block quantiser of the attention). The integer sums are exact, so a result depends neither on
the launch's shape nor on the batch a token is in. Rows of codes start on 16 bytes: with
``in_features`` not a multiple of 16 they are a view of wider rows, as
:func:`quantize_per_token_int8` allocates them. For inference: no gradient passes through.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor, nn

from tilemix_b200._lib import TM_DTYPE_BF16, TM_DTYPE_FP16, TM_DTYPE_FP32, launcher

__all__ = ["quantize_per_token_int8", "int8_matmul", "int8_linear", "Int8Linear"]

_DTYPES = {torch.float16: TM_DTYPE_FP16, torch.bfloat16: TM_DTYPE_BF16, torch.float32: TM_DTYPE_FP32}
_launch_quant, _launch_matmul = launcher("tm_quant_per_token_int8"), launcher("tm_int8_matmul")
_launch_linear = launcher("tm_int8_linear")


def quantize_per_token_int8(x: Tensor) -> tuple[Tensor, Tensor]:
    """Codes int8 [rows, cols] and scales fp32 [rows] of fp16 or bf16 ``x`` [rows, cols] (columns
    contiguous). A row of zeros has scale 0; a row with an infinity or a NaN has that scale."""
    codes, scale = _quantise(x)
    return (codes if codes.shape[1] == x.shape[1] else codes[:, :x.shape[1]]), scale


def _quantise(x: Tensor) -> tuple[Tensor, Tensor]:
    """:func:`quantize_per_token_int8` with the codes' rows as they are laid out, whole 16 bytes wide."""
    if not x.is_cuda:
        raise RuntimeError("the quantiser is a CUDA kernel")
    if x.ndim != 2 or x.shape[1] == 0:
        raise ValueError("expected [rows, cols] with at least one column")
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("the per-token quantiser takes fp16 or bf16")
    if x.stride(1) != 1 and x.shape[1] > 1:
        raise ValueError("the columns must be contiguous")
    rows, cols = x.shape
    codes = torch.empty((rows, (cols + 15) // 16 * 16), dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    _launch_quant(x.get_device(), x.data_ptr(), _DTYPES[x.dtype], x.stride(0), rows, cols,
                  codes.data_ptr(), codes.stride(0), scale.data_ptr())
    return codes, scale


def _check_weight(w8: Tensor, w_scale: Tensor, in_features: int, index: int) -> None:
    if w8.dtype is not torch.int8 or w_scale.dtype is not torch.float32:
        raise TypeError("codes must be torch.int8 and scales torch.float32")
    if w8.ndim != 2 or w_scale.ndim != 1:
        raise ValueError("expected codes [rows, in_features] and one scale a row")
    n, k = w8.shape
    if w_scale.shape[0] != n:
        raise ValueError("expected codes [rows, in_features] and one scale a row")
    if n == 0 or k == 0:
        raise ValueError("a linear layer needs at least one input and one output feature")
    if k != in_features:
        raise ValueError(f"in_features differ: {in_features} and {k}")
    if w8.get_device() != index or w_scale.get_device() != index:
        raise ValueError("all tensors of a call must share one CUDA device")
    _check_rows("w8", w8)
    if w_scale.stride(0) != 1 and n > 1:
        raise ValueError("scales must be contiguous")


def _check_rows(name: str, t: Tensor) -> None:
    if (t.stride(1) != 1 and t.shape[1] > 1) or t.data_ptr() % 16 or (t.shape[0] > 1 and t.stride(0) % 16):
        raise ValueError(f"{name} must have contiguous columns and rows that start on 16 bytes "
                         "(quantize_per_token_int8 lays them out so)")


def _check_bias(bias: Optional[Tensor], rows: int, dtype, index: int) -> None:
    if bias is None:
        return
    if bias.dtype != dtype:
        raise TypeError("the bias must have the output's dtype")
    if bias.shape != (rows,) or not bias.is_contiguous():
        raise ValueError("the bias must be contiguous with one value for each output feature")
    if bias.get_device() != index:
        raise ValueError("all tensors of a call must share one CUDA device")


def int8_matmul(x8: Tensor, x_scale: Tensor, w8: Tensor, w_scale: Tensor, bias: Optional[Tensor] = None, *,
                out_dtype: torch.dtype = torch.float16) -> Tensor:
    """``(x8 . w8^T) * x_scale[:, None] * w_scale + bias`` as ``out_dtype`` (fp16, bf16 or fp32), for
    codes ``x8`` [tokens, in_features] and ``w8`` [out_features, in_features] and fp32 scales."""
    if not x8.is_cuda:
        raise RuntimeError("the matrix product is a CUDA kernel")
    if out_dtype not in _DTYPES:
        raise TypeError("out_dtype must be float16, bfloat16 or float32")
    if x8.dtype != torch.int8 or x_scale.dtype != torch.float32:
        raise TypeError("codes must be torch.int8 and scales torch.float32")
    if x8.ndim != 2 or x_scale.ndim != 1 or x_scale.shape[0] != x8.shape[0] or not x_scale.is_contiguous():
        raise ValueError("expected codes [tokens, in_features] and one contiguous scale a token")
    if x_scale.get_device() != x8.get_device():
        raise ValueError("all tensors of a call must share one CUDA device")
    _check_weight(w8, w_scale, x8.shape[1], x8.get_device())
    _check_rows("x8", x8)
    _check_bias(bias, w8.shape[0], out_dtype, x8.get_device())
    out = torch.empty((x8.shape[0], w8.shape[0]), dtype=out_dtype, device=x8.device)
    _launch_matmul(x8.get_device(), x8.data_ptr(), x8.stride(0), x_scale.data_ptr(), w8.data_ptr(), w8.stride(0),
                   w_scale.data_ptr(), 0 if bias is None else bias.data_ptr(), out.data_ptr(), out.stride(0),
                   _DTYPES[out_dtype], x8.shape[0], w8.shape[0], x8.shape[1])
    return out


def int8_linear(x: Tensor, w8: Tensor, w_scale: Tensor, bias: Optional[Tensor] = None) -> Tensor:
    """A linear layer with its weight in 8 bits: ``x`` [..., in_features] (fp16 or bf16) is quantised by
    token, multiplied with ``w8`` [out_features, in_features] and returned in its own dtype."""
    if not x.is_cuda:
        raise RuntimeError("the linear layer is a CUDA kernel")
    if x.ndim == 0:
        raise ValueError("expected [..., in_features]")
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("the per-token quantiser takes fp16 or bf16")
    index, dtype, k = x.get_device(), x.dtype, x.shape[-1]
    _check_weight(w8, w_scale, k, index)
    n = w8.shape[0]
    _check_bias(bias, n, dtype, index)
    rows = x if x.ndim == 2 else x.reshape(-1, k)
    m = rows.shape[0]
    row_stride, column_stride = rows.stride()
    if column_stride != 1 and k > 1:
        rows, row_stride = rows.contiguous(), k
    out = x.new_empty((m, n))
    # One piece of scratch: the codes, their rows on 16 bytes, and behind them the scales.
    wide = (k + 15) // 16 * 16
    scratch = w8.new_empty(m * (wide + 4))
    codes = scratch.data_ptr()
    _launch_linear(index, rows.data_ptr(), _DTYPES[dtype], row_stride, codes, wide, codes + m * wide,
                   w8.data_ptr(), w8.stride(0), w_scale.data_ptr(), 0 if bias is None else bias.data_ptr(),
                   out.data_ptr(), n, m, n, k)
    return out if x.ndim == 2 else out.view(*x.shape[:-1], n)


class Int8Linear(nn.Module):
    """``nn.Linear`` for inference with the weight in 8 bits, one scale for each output feature. The
    codes are laid out once, rows on 16 bytes (buffer ``codes``); ``weight`` is their view. ``half()``,
    ``bfloat16()`` and ``to(dtype)`` change the activations' type and the bias; the scales stay fp32."""

    def __init__(self, linear: nn.Linear):
        super().__init__()
        if linear.weight.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("Int8Linear replaces an fp16 or bf16 linear layer")
        self.in_features, self.out_features = linear.in_features, linear.out_features
        self.dtype = linear.weight.dtype
        with torch.no_grad():
            codes, scale = _quantise(linear.weight.detach().contiguous())
        self.register_buffer("codes", codes)
        self.register_buffer("weight_scale", scale)
        self.register_buffer("bias", None if linear.bias is None else linear.bias.detach().clone())
        self.train(linear.training)

    @property
    def weight(self) -> Tensor:
        """The codes, int8 [out_features, in_features]."""
        return self.codes[:, :self.in_features]

    def _apply(self, fn, recurse=True):
        scale = self.weight_scale
        super()._apply(fn, recurse)
        if self.weight_scale.dtype != scale.dtype:
            self.weight_scale = scale.to(self.weight_scale.device)
        self.dtype = fn(torch.empty(0, dtype=self.dtype, device=scale.device)).dtype
        return self

    def forward(self, x: Tensor) -> Tensor:
        if x.dtype != self.dtype:
            raise TypeError(f"the layer takes {self.dtype} activations, got {x.dtype}")
        return int8_linear(x, self.weight, self.weight_scale, self.bias)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
