"""Layer norm over the last dimension, forward and backward, on B200 kernels.

    mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) r
    y = h * weight + bias
    with q = dy * weight:  dx = r (q - mean(q) - h mean(q h))
    dweight = sum over rows of dy h,  dbias = sum over rows of dy

`layer_norm` is the entry point; `torch.ops.tensorcore_gemm.layer_norm` is the
same operator for tracers (it also returns the rows' statistics).  Statistics
and sums are in fp32; each result is rounded once.  CUDA tensors only; nothing
falls back to another implementation.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _native
from ._rows import (DTYPE_CODES, as_rows, check_cuda, check_operand, launch, once_differentiable, plain_eager, ptr,
                    refuse_tangents, wants_grad, workspace)


def _check(x, weight, bias) -> None:
    check_cuda("x", x)
    if x.dim() < 1:
        raise RuntimeError("x must have at least one dimension")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        check_cuda(name, t, (x.dtype, torch.float32) if x.dtype != torch.float32 else (torch.float32,))
        if t.dim() != 1 or t.shape[0] != x.shape[-1]:
            raise RuntimeError(f"{name} must be 1-D with x's last dimension's size")
        if t.device != x.device:
            raise RuntimeError(f"{name} must be on x's device")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError("weight and bias must have the same dtype")


def _wdtype(x, weight, bias):
    return weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype


def _forward(x, weight, bias, eps: float, stats: bool):
    """y, and with `stats` the rows' mean and 1 / standard deviation (fp32, 2 x rows)."""
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    cols = x.shape[-1]
    rows = x.numel() // cols if cols else 0
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device) if stats else None
    if rows:
        x2, ldx = as_rows(x)
        weight = None if weight is None else weight.contiguous()
        bias = None if bias is None else bias.contiguous()
        mean = ptr(stats)
        launch("b200_layer_norm_fwd", x.get_device(), x2.data_ptr(), ptr(weight), ptr(bias), y.data_ptr(), mean,
               None if mean is None else mean + 4 * rows, rows, cols, ldx, cols, DTYPE_CODES[x.dtype],
               DTYPE_CODES[_wdtype(x, weight, bias)], eps)
    return y, stats


def _backward(dy, x, weight, stats, wdtype, need_weight: bool, need_bias: bool):
    """dx, dweight and dbias (None where not needed)."""
    cols = x.shape[-1]
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    dw = torch.empty(cols, dtype=wdtype, device=x.device) if need_weight else None
    db = torch.empty(cols, dtype=wdtype, device=x.device) if need_bias else None
    if cols:
        rows = x.numel() // cols
        x2, ldx = as_rows(x)
        dy2, lddy = as_rows(dy)
        weight = None if weight is None else weight.contiguous()
        mean = stats.data_ptr()
        ws_bytes = 0
        if need_weight or need_bias:
            ws_bytes = _native.load().b200_layer_norm_bwd_workspace_size(rows, cols)
        ws = workspace(ws_bytes, x.device, "b200_layer_norm_bwd_workspace_size")
        launch("b200_layer_norm_bwd", x.get_device(), dy2.data_ptr(), x2.data_ptr(), ptr(weight), mean,
               mean + 4 * rows, dx.data_ptr(), ptr(dw), ptr(db), rows, cols, lddy, ldx, cols, DTYPE_CODES[x.dtype],
               DTYPE_CODES[wdtype], ptr(ws), ws_bytes)
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.wdtype = _wdtype(x, weight, bias)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        if plain_eager(dy):
            dx, dw, db = _backward(dy, x, weight, stats, ctx.wdtype, need_w, need_b)
        else:
            dx, dw, db = torch.ops.tensorcore_gemm.layer_norm_backward(dy, x, weight, stats, ctx.wdtype, need_w, need_b)
        return dx if need_x else None, dw if need_w else None, db if need_b else None, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm of `x` (..., N) over its last dimension.

    x is float16, bfloat16 or float32; weight and bias (N each, optional) have
    x's type or float32.  Rows may be strided.  Differentiable in x, weight and
    bias (once).
    """
    if not plain_eager(x, weight, bias):
        return torch.ops.tensorcore_gemm.layer_norm(x, weight, bias, eps)[0]
    _check(x, weight, bias)
    if wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _forward(x, weight, bias, eps, False)[0]


# ---------------------------------------------------------------------------
# The dispatcher operators
# ---------------------------------------------------------------------------
@torch.library.custom_op("tensorcore_gemm::layer_norm", mutates_args=())
def _layer_norm_op(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor],
                   eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """y of `layer_norm`, and the rows' mean and 1 / standard deviation (not differentiable)."""
    _check(x, weight, bias)
    refuse_tangents(x, weight, bias)
    return _forward(x, weight, bias, eps, True)


@_layer_norm_op.register_fake
def _(x, weight, bias, eps):
    _check(x, weight, bias)
    rows = x.numel() // x.shape[-1] if x.shape[-1] else 0
    return (torch.empty(x.shape, dtype=x.dtype, device=x.device),
            torch.empty((2, rows), dtype=torch.float32, device=x.device))


@torch.library.custom_op("tensorcore_gemm::layer_norm_backward", mutates_args=())
def _layer_norm_backward_op(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], stats: torch.Tensor,
                            wdtype: torch.dtype, need_weight: bool = True,
                            need_bias: bool = True) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """dx, dweight and dbias (the latter two without elements where not needed)."""
    _check(x, weight, None)
    if wdtype not in (x.dtype, torch.float32) or (weight is not None and weight.dtype != wdtype):
        raise RuntimeError("wdtype must be weight's dtype, and x's or float32")
    dy = check_operand("dy", dy, x.shape, x.dtype, x.device)
    rows = x.numel() // x.shape[-1] if x.shape[-1] else 0
    stats = check_operand("stats", stats, (2, rows), torch.float32, x.device)
    grads = _backward(dy, x, weight, stats, wdtype, need_weight, need_bias)
    return tuple(x.new_empty(0, dtype=wdtype) if g is None else g for g in grads)


@_layer_norm_backward_op.register_fake
def _(dy, x, weight, stats, wdtype, need_weight=True, need_bias=True):
    sums = [torch.empty(x.shape[-1] if need else 0, dtype=wdtype, device=x.device) for need in (need_weight, need_bias)]
    return torch.empty(x.shape, dtype=x.dtype, device=x.device), *sums


def _setup_context(ctx, inputs, output) -> None:
    x, weight, bias, _ = inputs
    ctx.save_for_backward(x, weight, output[1])
    ctx.wdtype = _wdtype(x, weight, bias)
    ctx.mark_non_differentiable(output[1])


def _op_backward(ctx, dy, _dstats):
    x, weight, stats = ctx.saved_tensors
    need_x, need_w, need_b, _ = ctx.needs_input_grad
    dx, dw, db = torch.ops.tensorcore_gemm.layer_norm_backward(dy, x, weight, stats, ctx.wdtype, need_w, need_b)
    return dx if need_x else None, dw if need_w else None, db if need_b else None, None


_layer_norm_op.register_autograd(_op_backward, setup_context=_setup_context)
