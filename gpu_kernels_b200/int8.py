"""Int8 on the GPU, with a scale for each token and each output channel: quantise, products, products expert by expert.

Beside the NVFP4 path, for weights that are kept in 8 bits. `quantize_int8` gives a matrix [rows, K] its codes and one
scale per row, for activations (a row is a token) and weights (a row is an output channel) alike; `int8_gemm` multiplies
two such matrices, `int8_linear` quantises the activations on the way, and `int8_grouped_gemm` multiplies rows sorted by
expert (`gather_tokens_int8`) with the expert's own weights. The sums are exact 32-bit integers, the scaling is FP32.
Nothing here has a gradient. Operands may have any strides and alignment, but one that is not contiguous or not on a 16-byte
boundary is copied whole on every call (weights too, of all experts): keep weights contiguous, as torch allocates them. An
`out` has to be contiguous and on a 16-byte boundary. The work is done by csrc/int8_quant.cu and csrc/int8_gemm.cu through the C ABI
(include/operators_capi.h); CPU tensors are rejected. Everything is asynchronous on the current stream, may be captured
into a CUDA graph and keeps nothing between calls; `check_int8` reports a product that gave up waiting inside the kernel.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .nvfp4 import _DTYPES, _require_cuda

MAX_K = 131056              # the sum of K products of int8 codes fits 32 bits


def matrix(rows: int, columns: int, dtype: torch.dtype, device) -> torch.Tensor:
    # (torch.empty takes 0.9 us longer: a tenth of a small call)
    return torch.empty_strided((rows, columns), (columns, 1), dtype=dtype, device=device)


def placed(t: torch.Tensor):
    """(t, its address), t contiguous and on a 16-byte boundary: as it is where it is that already, else a copy."""
    if not t.is_contiguous():
        t = t.contiguous()
    address = t.data_ptr()
    if address % 16:
        t = t.clone()
        address = t.data_ptr()
    return t, address


def _rows(values: torch.Tensor, name: str):
    _require_cuda(values, name)
    if values.dim() != 2:
        raise ValueError(f"{name} must be 2-D [rows, K]")
    if values.dtype not in _DTYPES:
        values = values.float()
    return placed(values.detach() if values.requires_grad else values)


def quantize_int8(values: torch.Tensor):
    """[rows, K] (bf16, fp16 or fp32; any K below 2^31) -> (codes int8 [rows, K], scales fp32 [rows]).

    scale = max|row| / 127; a code is the integer nearest to 127 * value / max|row|, ties to the even one. A zero row has
    scale 0; a row that holds a NaN or an infinity has scale NaN and codes 0, so that what is computed from it is NaN."""
    values, address = _rows(values, "values")
    rows, k = values.shape
    if k >> 31:
        raise ValueError("K must be below 2^31")
    device = values.device
    codes = matrix(rows, k, torch.int8, device)
    scales = torch.empty(rows, dtype=torch.float32, device=device)
    _lib.run(device, _lib.load().gpu_kernels_int8_quantize, address, _DTYPES[values.dtype], codes.data_ptr(), scales.data_ptr(), rows, k)
    return codes, scales


def dequantize_int8(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """codes * scales[:, None] -> fp32 [rows, K]."""
    _operand(codes, "codes", 2)
    codes, at_codes = placed(codes)
    rows, k = codes.shape
    if k >> 31:
        raise ValueError("K must be below 2^31")
    device = codes.device
    scales, at_scales = _scales(scales, "scales", (rows,), device)
    out = matrix(rows, k, torch.float32, device)
    _lib.run(device, _lib.load().gpu_kernels_int8_dequantize, at_codes, at_scales, out.data_ptr(), rows, k)
    return out


def _operand(t: torch.Tensor, name: str, dim: int, device=None) -> None:
    if not (t.is_cuda and t.dtype == torch.int8 and t.dim() == dim):
        raise ValueError(f"{name} must be a {dim}-D CUDA int8 tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name} must be on {device}, where the other operands are")


def _scales(t: torch.Tensor, name: str, shape, device):
    if t.dtype != torch.float32 or t.shape != shape or t.device != device:
        raise ValueError(f"{name} must be an fp32 tensor of shape {tuple(shape)} on {device}")
    return placed(t)


def _output(out, m, n, dtype, device) -> torch.Tensor:
    if out is None:
        if dtype not in _DTYPES:
            raise ValueError("out_dtype must be bf16, fp16 or fp32")
        return matrix(m, n, dtype, device)
    if not (out.device == device and out.dtype in _DTYPES and out.is_contiguous() and out.shape == (m, n)):
        raise ValueError(f"out must be a contiguous bf16, fp16 or fp32 tensor of shape {(m, n)} on {device}")
    return out


def _check_sizes(m: int, n: int, k: int, other_k: int) -> None:
    if k != other_k:
        raise ValueError("the operands disagree on K")
    if m > 1 << 30 or n > 1 << 30:
        raise ValueError("M and N up to 2^30")
    if n < 8 or n % 8 or k < 16 or k % 16 or k > MAX_K:
        raise ValueError(f"N must be a multiple of 8 and K a multiple of 16 up to {MAX_K}")


def int8_gemm(a: torch.Tensor, b: torch.Tensor, a_scales: torch.Tensor, b_scales: torch.Tensor, out: torch.Tensor | None = None,
              out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """C [M, N] = (a [M, K] @ b [N, K].T) * a_scales[:, None] * b_scales, in out's type (or out_dtype).

    M and N up to 2^30; N a multiple of 8, K a multiple of 16 up to 131056."""
    device = a.device
    _operand(a, "a", 2)
    _operand(b, "b", 2, device)
    (m, k), (n, k2) = a.shape, b.shape
    _check_sizes(m, n, k, k2)
    (a, at_a), (b, at_b) = placed(a), placed(b)
    a_scales, at_a_scales = _scales(a_scales, "a_scales", (m,), device)
    b_scales, at_b_scales = _scales(b_scales, "b_scales", (n,), device)
    out = _output(out, m, n, out_dtype, device)
    _lib.run(device, _lib.load().gpu_kernels_int8_gemm, at_a, at_b, at_a_scales, at_b_scales, out.data_ptr(), _DTYPES[out.dtype], m, n, k)
    return out


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor, out: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """x [M, K] (bf16, fp16 or fp32), quantised token by token, times weight [N, K] int8 -> [M, N] in x's type (or
    out_dtype): int8_gemm(*quantize_int8(x), ...) in one call. The product requests its first weights while the quantiser
    runs."""
    x, at_x = _rows(x, "x")
    device, dtype = x.device, x.dtype
    _operand(weight, "weight", 2, device)
    (m, k), (n, k2) = x.shape, weight.shape
    _check_sizes(m, n, k, k2)
    weight, at_weight = placed(weight)
    weight_scales, at_scales = _scales(weight_scales, "weight_scales", (n,), device)
    out = _output(out, m, n, out_dtype or dtype, device)
    room = torch.empty(m * (k + 4), dtype=torch.uint8, device=device)               # the codes, then the tokens' scales
    codes = room.data_ptr()
    _lib.run(device, _lib.load().gpu_kernels_int8_linear, at_x, _DTYPES[dtype], at_weight, at_scales, codes, codes + m * k,
             out.data_ptr(), _DTYPES[out.dtype], m, n, k)
    return out


def int8_grouped_gemm(rows: torch.Tensor, weights: torch.Tensor, row_scales: torch.Tensor, weight_scales: torch.Tensor,
                      offsets: torch.Tensor, out: torch.Tensor | None = None,
                      out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """rows [R, K] sorted by expert, weights [E, N, K] -> C [R, N]: the rows [offsets[e], offsets[e + 1]) times weights[e].

    offsets int32 [E + 1] as `sort_routes` gives them; they stay on the GPU. Rows of no expert (at or behind offsets[E], in front of offsets[0])
    are zeros in a C made here and are left as they were in an `out` that is handed in. E up to 1024; N and K as in
    int8_gemm."""
    _operand(rows, "rows", 2)
    _operand(weights, "weights", 3, rows.device)
    (r, k), (experts, n, k2) = rows.shape, weights.shape
    _check_sizes(r, n, k, k2)
    if not 1 <= experts <= 1024:
        raise ValueError("1..1024 experts")
    if offsets.dtype != torch.int32 or offsets.shape != (experts + 1,) or offsets.device != rows.device:
        raise ValueError(f"offsets must be an int32 tensor of {experts + 1} values on {rows.device}")
    device = rows.device
    (rows, at_rows), (weights, at_weights), offsets = placed(rows), placed(weights), offsets.contiguous()
    row_scales, at_row_scales = _scales(row_scales, "row_scales", (r,), device)
    weight_scales, at_weight_scales = _scales(weight_scales, "weight_scales", (experts, n), device)
    made = out is None
    out = _output(out, r, n, out_dtype, device)
    _lib.run(device, _lib.load().gpu_kernels_int8_grouped_gemm, at_rows, at_weights, at_row_scales, at_weight_scales,
             offsets.data_ptr(), experts, out.data_ptr(), _DTYPES[out.dtype], r, n, k, 1 if made else 0)
    return out


def int8_tiles(rows: int, n: int, k: int, experts: int = 0) -> dict:
    """What a product of these sizes runs on the current device (experts > 0: a grouped one)."""
    if max(rows, n, k, experts) >> 31:
        raise ValueError("sizes of fewer than 32 bits")
    info = (ctypes.c_int * 5)()
    _lib.check(_lib.load().gpu_kernels_int8_tiles(rows, n, k, experts, info))
    return dict(zip(("pair", "swap", "width", "split", "stages"), info))


def check_int8(device=None) -> None:
    """Synchronises and raises if a product on this device gave up waiting inside the kernel since the last check."""
    with torch.cuda.device(device):
        _lib.check(_lib.load().gpu_kernels_nvfp4_validate(None))
