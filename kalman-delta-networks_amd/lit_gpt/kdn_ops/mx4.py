"""Microscaled 4-bit matrices (MX4) and the linear product with MX4 weights, for serving.

The reference has no counterpart: its models run in bf16 and fp32.  A decode step is bound by the weight stream, and
an MX4 weight is 4.25 bits an element where bf16 has 16.

A row of K elements is held in groups of 128: 64 bytes of codes (E2M1, two to a byte, the lower nibble first) and 4
scale bytes, one per block of 32 elements, s standing for 2^(s - 127) (255: NaN).  The padding past K is zero.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch

from . import _lib

GROUP = 128
MAX_ROW_STRIDE = 1 << 21  # of bf16 x, in elements: kdn_mx4_linear addresses a tile's rows by 32-bit offsets


class MX4Tensor(NamedTuple):
    """A matrix [rows, cols] in MX4: ``codes`` uint8 [rows, 64 G], ``scales`` uint8 [rows, 4 G], G = ceil(cols / 128)."""
    codes: torch.Tensor
    scales: torch.Tensor
    cols: int

    @property
    def rows(self) -> int:
        return self.codes.shape[0]


# A decode step's products take 5 to 8 us on the GPU, so the checks around a launch are kept short: the host takes 9.2 us
# for one of them (the launch 3.4, the output 1.7); with a generic device check, generator expressions and the workspace
# query it took 10.5.
def _check(name: str, t: MX4Tensor) -> int:
    if type(t) is not MX4Tensor:
        raise TypeError(f"{name} must be an MX4Tensor, got {type(t).__name__}")
    codes, scales, cols = t
    if codes.dtype is not torch.uint8 or scales.dtype is not torch.uint8:
        raise TypeError(f"{name}: codes and scales must be uint8, got {codes.dtype} and {scales.dtype}")
    groups = -(-cols // GROUP)
    rows = codes.shape[0] if codes.ndim else 0
    if cols < 1 or codes.shape != (rows, 64 * groups) or scales.shape != (rows, 4 * groups):
        raise ValueError(f"{name}: {cols} columns take codes [rows, {64 * groups}] and scales [rows, {4 * groups}], got "
                         f"{tuple(codes.shape)} and {tuple(scales.shape)}")
    if not (codes.is_contiguous() and scales.is_contiguous()) or codes.data_ptr() % 16 or scales.data_ptr() % 4:
        raise ValueError(f"{name}: codes must be contiguous and 16-byte aligned, scales contiguous and 4-byte aligned")
    return rows


def mx4_quantize(x: torch.Tensor) -> MX4Tensor:
    """``x`` [..., K] (bf16 or fp32) in MX4, its leading dimensions as rows.

    Per block of 32 elements the scale puts the largest magnitude into [4, 8) units; every element goes to the nearest
    of 0, 0.5, 1, 1.5, 2, 3, 4, 6 units (ties to the even code), larger ones to 6.  A block that holds an infinity or
    NaN is NaN."""
    if x.dtype != torch.bfloat16 and x.dtype != torch.float32:
        raise TypeError(f"x must be bf16 or fp32, got {x.dtype}")
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have at least one column, got {tuple(x.shape)}")
    _lib.refuse_derivatives("mx4_quantize", x)
    _lib.one_device(x)
    K = x.shape[-1]
    x2 = x if x.ndim == 2 else x.reshape(-1, K)
    rows, groups = x2.shape[0], -(-K // GROUP)
    if (K > 1 and x2.stride(1) != 1) or (rows > 1 and x2.stride(0) < K):
        x2 = x2.contiguous()
    codes = torch.empty((rows, 64 * groups), device=x.device, dtype=torch.uint8)
    scales = torch.empty((rows, 4 * groups), device=x.device, dtype=torch.uint8)
    if rows:
        with _lib.on(x.device):
            _lib.call("kdn_mx4_quantize", x2.data_ptr(), _lib.is_bf16(x2), x2.stride(0), rows, K, codes.data_ptr(),
                      scales.data_ptr(), _lib.stream_of(x2))
    return MX4Tensor(codes, scales, K)


def mx4_dequantize(t: MX4Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values [rows, cols] that ``t`` stands for, in fp32 or bf16: both hold every value that
    ``mx4_quantize`` gives (a block of its scales reaches 2^125; foreign scales past that may overflow)."""
    rows = _check("t", t)
    if dtype != torch.bfloat16 and dtype != torch.float32:
        raise TypeError(f"dtype must be bf16 or fp32, got {dtype}")
    _lib.one_device(t.codes, t.scales)
    y = torch.empty((rows, t.cols), device=t.codes.device, dtype=dtype)
    if rows:
        with _lib.on(y.device):
            _lib.call("kdn_mx4_dequantize", t.codes.data_ptr(), t.scales.data_ptr(), rows, t.cols, y.data_ptr(),
                      _lib.is_bf16(y), _lib.stream_of(y))
    return y


def mx4_linear(x: Union[torch.Tensor, MX4Tensor], weight: MX4Tensor, bias: Optional[torch.Tensor] = None, *,
               residual: Optional[torch.Tensor] = None, gated: bool = False) -> torch.Tensor:
    """[residual +] ``x`` @ ``weight``^T [+ bias] in bf16, with fp32 sums and one rounding.

    ``x`` [..., K] bf16 is multiplied as it is (only the weights are rounded to 4 bits); an MX4Tensor [M, K] is
    multiplied in 4 bits on both sides.  ``gated``: ``weight`` [2N, K] = [w1; w2] and the result is the SwiGLU gate
    silu(x w1^T + b1) * (x w2^T + b2).  ``bias`` [N] ([2N] gated) and ``residual`` [..., N] are bf16."""
    R = _check("weight", weight)
    K = weight.cols
    if gated and R % 2:
        raise ValueError(f"a gated product takes a packed [2N, K] weight, got {R} rows")
    N = R // 2 if gated else R
    quantized = type(x) is MX4Tensor
    if quantized:
        M = _check("x", x)
        lead = (M,)
        x2, x_scales, row_stride = x.codes, x.scales, 0
        if x.cols != K:
            raise ValueError(f"x has {x.cols} columns, the weight {K}")
    else:
        if x.dtype != torch.bfloat16:
            raise TypeError(f"x must be bf16 or an MX4Tensor, got {x.dtype}")
        if x.ndim < 1 or x.shape[-1] != K:
            raise ValueError(f"x must have {K} columns, got {tuple(x.shape)}")
        lead = x.shape[:-1]
        x2 = x if x.ndim == 2 else x.reshape(-1, K)
        M, x_scales = x2.shape[0], None
    if bias is not None and (bias.dtype != torch.bfloat16 or bias.shape != (R,) or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous bf16 [{R}] or None")
    if residual is not None and (residual.dtype != torch.bfloat16 or residual.shape != (*lead, N)):
        raise ValueError(f"residual must be bf16 {(*lead, N)}, got {residual.dtype} {tuple(residual.shape)}")
    _lib.refuse_derivatives("mx4_linear", x2, bias, residual)
    _lib.one_device(x2, x_scales, weight.codes, weight.scales, bias, residual)
    res_stride = 0
    if residual is not None:
        residual = residual if residual.ndim == 2 else residual.reshape(M, N)
        if (N > 1 and residual.stride(1) != 1) or (M > 1 and residual.stride(0) < N):
            residual = residual.contiguous()
        res_stride = residual.stride(0)
    K8 = K
    if not quantized:
        # the kernels load 16-byte pieces of rows: rows of another length or alignment, or too far apart, are copied
        if K % 8:
            K8 = K + -K % 8
            padded = x2.new_zeros((M, K8))
            padded[:, :K] = x2
            x2 = padded
        elif x2.stride(1) != 1 or x2.data_ptr() % 16 or (M > 1 and (not K <= x2.stride(0) <= MAX_ROW_STRIDE
                                                                    or x2.stride(0) % 8)):
            x2 = x2.clone(memory_format=torch.contiguous_format)
        row_stride = x2.stride(0)
    y = torch.empty((*lead, N), device=x2.device, dtype=torch.bfloat16)
    if M and N:
        ws_bytes = _lib.size("kdn_mx4_linear_workspace_size", M, N, K8, int(quantized), int(gated)) if M > 16 else 0
        ws = torch.empty(ws_bytes, device=y.device, dtype=torch.uint8) if ws_bytes else None
        with _lib.on(y.device):
            _lib.call("kdn_mx4_linear", x2.data_ptr(), _lib.ptr(x_scales), row_stride, weight.codes.data_ptr(),
                      weight.scales.data_ptr(), _lib.ptr(bias), _lib.ptr(residual), res_stride, M, N, K8, int(gated),
                      y.data_ptr(), N, _lib.ptr(ws), ws_bytes, _lib.stream_of(y))
    return y


__all__ = ("MX4Tensor", "mx4_quantize", "mx4_dequantize", "mx4_linear")
