"""Tokens to their experts' rows and back, with gradients: what stands around an expert layer's products.

A router gives each token topk experts (`route`); a route is one of these choices. `sort_routes` orders the routes by
expert, `gather_tokens` copies the tokens' rows into that order (`gather_tokens_int8` quantises them on the way),
`combine_tokens` adds the experts' rows up again, weighted, token by token. `gather_tokens` and `combine_tokens` have
gradients, and refuse tensors with a forward-mode tangent; codes have neither. The order is stable and every sum is taken in
the order of the routes, so results do not change from run to run. The work is done by csrc/tokens.cu and
csrc/int8_quant.cu through the C ABI (include/operators_capi.h); CPU tensors are rejected. Everything is asynchronous on the
current stream and may be captured into a CUDA graph; nothing reads the routes back to the host.
(Capture a backward pass with leaves that no graph outside the capture still refers to: autograd accumulates into a leaf
on the stream where it was first used.)
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .int8 import matrix, placed
from .nvfp4 import _DTYPES, _require_cuda


class Routes(NamedTuple):
    """The order of a batch's routes: offsets int32 [E + 1] (expert e's rows are [offsets[e], offsets[e + 1])), position
    int32 [T, topk] (each route's row) and source int32 [T * topk] (each row's route, token * topk + choice). Routes of no
    expert have the rows from offsets[E] on.

    An order of a caller's own making has to be one too: every row the place of exactly one route. With others nothing is read
    or written out of bounds, but a row that no position names is not written, and one that several name is written by each."""
    offsets: torch.Tensor
    position: torch.Tensor
    source: torch.Tensor


def sort_routes(ids: torch.Tensor, num_experts: int) -> Routes:
    """ids [T, topk] (int64 or int32): the experts each token goes to. Rows are ordered by expert and, inside an expert, by
    token; an id outside [0, num_experts) (a router's "dropped" mark such as -1) belongs to no expert. Up to 1024 experts."""
    _require_cuda(ids, "ids")
    if ids.dim() != 2 or ids.dtype not in (torch.int64, torch.int32):
        raise ValueError("ids must be an int64 or int32 tensor [tokens, topk]")
    if not 1 <= num_experts <= 1024:
        raise ValueError("1..1024 experts")
    ids = ids.contiguous()
    routes, d = ids.numel(), ids.device
    if routes >= 1 << 31:
        raise ValueError("fewer than 2^31 routes")
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=d)
    position = matrix(*ids.shape, torch.int32, d)
    source = torch.empty(routes, dtype=torch.int32, device=d)
    lib = _lib.load()
    needed = lib.gpu_kernels_tokens_sort_workspace(routes, num_experts)
    room = torch.empty(needed, dtype=torch.uint8, device=d) if needed else None
    _lib.run(d, lib.gpu_kernels_tokens_sort, ids.data_ptr(), ids.element_size(), routes, num_experts, offsets.data_ptr(),
             position.data_ptr(), source.data_ptr(), None if room is None else room.data_ptr())
    return Routes(offsets, position, source)


def _places(position: torch.Tensor, offsets: torch.Tensor) -> tuple[int, int, int, int]:
    """The addresses of the positions and of the number of live rows, tokens, topk."""
    return (position.data_ptr(), offsets.data_ptr() + 4 * (offsets.numel() - 1), *position.shape)


def _check_routes(routes: Routes, tokens: int | None, device) -> tuple[int, int, int, int]:
    """The places of a checked order."""
    offsets, position = routes.offsets, routes.position
    shape = position.shape
    if len(shape) != 2 or shape[1] < 1 or (tokens is not None and shape[0] != tokens):
        raise ValueError("the routes are not those of this many tokens")
    batch, topk = shape
    if batch * topk >> 31:
        raise ValueError("fewer than 2^31 routes")
    for t in (offsets, position):
        if t.dtype != torch.int32 or t.device != device or not t.is_contiguous():
            raise ValueError(f"routes.{'offsets' if t is offsets else 'position'} must be a contiguous int32 tensor on {device}")
    if offsets.dim() != 1 or offsets.numel() < 2:
        raise ValueError("routes.offsets must hold one value per expert and one more")
    return position.data_ptr(), offsets.data_ptr() + 4 * (offsets.numel() - 1), batch, topk


def _values(t: torch.Tensor, name: str) -> torch.Tensor:
    _require_cuda(t, name)
    if t.dim() != 2 or t.dtype not in _DTYPES or not 1 <= t.shape[1] < 1 << 31:
        raise ValueError(f"{name} must be a bf16, fp16 or fp32 tensor [rows, hidden], hidden below 2^31")
    return t


def _gather(x, places):
    x = x.contiguous()
    position, live, tokens, topk = places
    hidden = x.shape[1]
    rows = matrix(tokens * topk, hidden, x.dtype, x.device)
    _lib.run(x.device, _lib.load().gpu_kernels_tokens_gather, x.data_ptr(), _DTYPES[x.dtype], tokens, topk, hidden, position, live,
             rows.data_ptr())
    return rows


def _combine(rows, places, weights):
    rows = rows.contiguous()
    position, live, tokens, topk = places
    hidden = rows.shape[1]
    y = matrix(tokens, hidden, rows.dtype, rows.device)
    _lib.run(rows.device, _lib.load().gpu_kernels_tokens_combine, rows.data_ptr(), _DTYPES[rows.dtype],
             None if weights is None else weights.data_ptr(), position, live, tokens, topk, hidden, y.data_ptr())
    return y


def _tangent(*tensors) -> bool:
    """Whether one of them has a tangent: the autograd functions then refuse the call."""
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


class _GatherTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, position, offsets, places):
        ctx.save_for_backward(position, offsets)
        return _gather(x, places)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_rows):
        # What hooks (save_on_cpu, checkpointing) give back belongs to this call alone: held by name until the launch, which
        # is given addresses.
        position, offsets = ctx.saved_tensors
        return _combine(d_rows, _places(position, offsets), None), None, None, None


class _CombineTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, position, offsets, places):
        ctx.save_for_backward(position, offsets, weights, rows if weights is not None and ctx.needs_input_grad[1] else None)
        return _combine(rows, places, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_y):
        position, offsets, weights, rows = ctx.saved_tensors                # (held until the launch, as above)
        places = _places(position, offsets)
        if weights is None:
            return _gather(d_y, places), None, None, None, None
        at_position, live, tokens, topk = places
        d_y = d_y.contiguous()
        hidden = d_y.shape[1]
        d_rows = d_weights = None
        if ctx.needs_input_grad[0]:
            d_rows = matrix(tokens * topk, hidden, d_y.dtype, d_y.device)
        if ctx.needs_input_grad[1]:
            d_weights = matrix(tokens, topk, torch.float32, d_y.device)
            rows = rows.contiguous()
        _lib.run(d_y.device, _lib.load().gpu_kernels_tokens_combine_backward, d_y.data_ptr(), _DTYPES[d_y.dtype],
                 None if rows is None else rows.data_ptr(), weights.data_ptr(), at_position, live, tokens, topk, hidden,
                 None if d_rows is None else d_rows.data_ptr(), None if d_weights is None else d_weights.data_ptr())
        return d_rows, d_weights, None, None, None


def gather_tokens(x: torch.Tensor, routes: Routes) -> torch.Tensor:
    """x [T, H] -> rows [T * topk, H]: each route's row is its token's. Rows of no expert are zeros.

    Gradient: x's is the sum of its live rows' gradients, in FP32 and the order of the routes, rounded once."""
    _values(x, "x")
    places = _check_routes(routes, x.shape[0], x.device)
    if x.requires_grad and torch.is_grad_enabled() or forward_ad._current_level >= 0 and _tangent(x):
        return _GatherTokens.apply(x, routes.position, routes.offsets, places)
    return _gather(x, places)


def gather_tokens_int8(x: torch.Tensor, routes: Routes):
    """quantize_int8(x) in the order of the routes: x [T, K] -> (codes int8 [T * topk, K], scales fp32 [T * topk]), the rows
    `int8_grouped_gemm` takes. A token is quantised once, K a multiple of 16; rows of no expert have codes and scale 0."""
    x, at_x = placed(_values(x, "x"))
    position, live, tokens, topk = _check_routes(routes, x.shape[0], x.device)
    k = x.shape[1]
    if k % 16:
        raise ValueError("K must be a multiple of 16")
    codes = matrix(tokens * topk, k, torch.int8, x.device)
    scales = torch.empty(tokens * topk, dtype=torch.float32, device=x.device)
    _lib.run(x.device, _lib.load().gpu_kernels_tokens_gather_int8, at_x, _DTYPES[x.dtype], tokens, topk, k, position, live,
             codes.data_ptr(), scales.data_ptr())
    return codes, scales


def combine_tokens(rows: torch.Tensor, routes: Routes, weights: torch.Tensor | None = None) -> torch.Tensor:
    """rows [T * topk, H], weights [T, topk] -> y [T, H]: the sum over a token's live routes of weight * row (None: of the
    rows), in FP32 and the order of the routes, rounded once. Rows of no expert are not read, whatever they hold.

    Gradients: a live row's is weight * d_y of its token, a weight's is <d_y, row>; zero for routes of no expert."""
    _values(rows, "rows")
    if rows.shape[0] != routes.position.numel():
        raise ValueError("the routes are not those of this many rows")
    if weights is not None:
        if weights.shape != routes.position.shape or weights.device != rows.device or not weights.is_floating_point():
            raise ValueError("weights must be floating-point, [tokens, topk] and where the rows are")
        weights = weights.float().contiguous()
    places = _check_routes(routes, None, rows.device)
    if (torch.is_grad_enabled() and (rows.requires_grad or (weights is not None and weights.requires_grad))
            or forward_ad._current_level >= 0 and _tangent(rows, weights)):
        return _CombineTokens.apply(rows, weights, routes.position, routes.offsets, places)
    return _combine(rows, places, weights)
