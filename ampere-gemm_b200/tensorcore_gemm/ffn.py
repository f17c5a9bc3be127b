"""Gated feed-forward block, forward and backward, on B200 kernels.

    g = x Wg^T, u = x Wu^T, a = act(g) u, y = a w_out^T        w_in = [Wg; Wu]
    da = dy w_out, dg = da u act'(g), du = da act(g)
    dx = [dg du] w_in, dw_in = [dg du]^T x, dw_out = dy^T a

Both input projections, the activation and the product are one launch, the
output projection a second one; so is da with dg, du and a in the backward
pass.  `gated_ffn` is the entry point; `torch.ops.tensorcore_gemm.gated_ffn`
is the same operator for tracers (it also returns [g u], without rows where
its `save` is false).  fp16 or bf16
operands, fp32 accumulation and activation; CUDA tensors only, nothing falls
back to another implementation.
"""
from __future__ import annotations

import torch

from . import _native
from ._rows import (DTYPE_CODES, as_rows, check_cuda, check_operand, launch, once_differentiable, plain_eager, ptr,
                    refuse_tangents, wants_grad, workspace)

ACTIVATIONS = {"silu": _native.B200_ACT_SILU, "gelu": _native.B200_ACT_GELU, "gelu_tanh": _native.B200_ACT_GELU_TANH}

_TYPES = (torch.float16, torch.bfloat16)


def _check(x, w_in, w_out, activation) -> None:
    if activation not in ACTIVATIONS:
        raise ValueError(f"Unsupported activation {activation!r}. Expected one of {tuple(ACTIVATIONS)}.")
    for name, t in (("x", x), ("w_in", w_in), ("w_out", w_out)):
        check_cuda(name, t, _TYPES)
        if t.dtype != x.dtype:
            raise RuntimeError(f"{name} must have x's dtype")
        if t.device != x.device:
            raise RuntimeError("x, w_in and w_out must be on the same CUDA device")
    if x.dim() < 1 or w_in.dim() != 2 or w_out.dim() != 2:
        raise RuntimeError("x needs at least one dimension, w_in and w_out two")
    if w_in.shape[1] != x.shape[-1]:
        raise RuntimeError("Inner dimensions must match: w_in is 2F x D for x of width D")
    if w_in.shape[0] != 2 * w_out.shape[1]:
        raise RuntimeError("w_in must have twice as many rows (gate, then up) as w_out has columns")


def _pad8(n: int) -> int:
    return -(-n // 8) * 8


def _unaligned(pointers: int, pitches: int) -> int:
    """1 when the rows of some operand do not start on 16 bytes, from the operands' addresses and pitches or-ed."""
    return 1 if pointers % 16 or pitches % 8 else 0


def _forward(x, w_in, w_out, activation: str, save: bool):
    """y, and with `save` [g u] (rows x 2 hidden, each half padded to a multiple of 8) for the backward pass."""
    dim, (out_dim, hidden) = x.shape[-1], w_out.shape
    rows = x.numel() // dim if dim else x.shape[:-1].numel()
    gate_up = torch.empty((rows, 2 * _pad8(hidden)), dtype=x.dtype, device=x.device) if save else None
    if rows == 0 or out_dim == 0 or dim == 0 or hidden == 0:
        return x.new_zeros((*x.shape[:-1], out_dim)), gate_up
    x2, ldx = as_rows(x)
    wi, ldi = as_rows(w_in)
    wo, ldo = as_rows(w_out)
    y = torch.empty((*x.shape[:-1], out_dim), dtype=x.dtype, device=x.device)
    xp, wip, wop, yp = x2.data_ptr(), wi.data_ptr(), wo.data_ptr(), y.data_ptr()
    ws_bytes = _native.load().b200_gated_ffn_workspace_size(
        rows, dim, hidden, out_dim, 0, _unaligned(xp | wip | wop | yp, ldx | ldi | ldo | out_dim))
    ws = workspace(ws_bytes, x.device, "b200_gated_ffn_workspace_size")
    launch("b200_gated_ffn_fwd", x.get_device(), xp, wip, wop, yp, ptr(gate_up), rows, dim, hidden,
           out_dim, ldx, ldi, ldo, out_dim, ACTIVATIONS[activation], DTYPE_CODES[x.dtype], ptr(ws), ws_bytes)
    return y, gate_up


def _backward(dy, x, w_in, w_out, gate_up, activation: str, need_x: bool, need_in: bool, need_out: bool):
    """dx, dw_in and dw_out (None where not needed)."""
    dim, (out_dim, hidden) = x.shape[-1], w_out.shape
    rows = gate_up.shape[0]
    new = torch.zeros_like if rows == 0 or out_dim == 0 or dim == 0 or hidden == 0 else torch.empty_like
    dx, dwi, dwo = (new(t, memory_format=torch.contiguous_format) if need else None
                    for t, need in ((x, need_x), (w_in, need_in), (w_out, need_out)))
    if new is torch.zeros_like:
        return dx, dwi, dwo
    dy2, lddy = as_rows(dy)
    x2, ldx = as_rows(x)
    wi, ldi = as_rows(w_in)
    wo, ldo = as_rows(w_out)
    dyp, xp, wip, wop = dy2.data_ptr(), x2.data_ptr(), wi.data_ptr(), wo.data_ptr()
    ws_bytes = _native.load().b200_gated_ffn_workspace_size(
        rows, dim, hidden, out_dim, 1, _unaligned(dyp | xp | wip | wop, lddy | ldx | ldi | ldo))
    ws = workspace(ws_bytes, x.device, "b200_gated_ffn_workspace_size")
    launch("b200_gated_ffn_bwd", x.get_device(), dyp, xp, wip, wop, gate_up.data_ptr(), ptr(dx), ptr(dwi), ptr(dwo),
           rows, dim, hidden, out_dim, lddy, ldx, ldi, ldo, dim, dim, hidden, ACTIVATIONS[activation],
           DTYPE_CODES[x.dtype], ptr(ws), ws_bytes)
    return dx, dwi, dwo


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_in, w_out, activation):
        y, gate_up = _forward(x, w_in, w_out, activation, True)
        ctx.save_for_backward(x, w_in, w_out, gate_up)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        if plain_eager(dy):
            return *_backward(dy, *ctx.saved_tensors, ctx.activation, *ctx.needs_input_grad[:3]), None
        return *_traced_backward(dy, ctx.saved_tensors, ctx.activation, ctx.needs_input_grad), None


def gated_ffn(x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """y = (act(x Wg^T) * (x Wu^T)) w_out^T for x (..., D), w_in = [Wg; Wu] (2F x D) and w_out (N x F).

    All float16 or all bfloat16.  activation: "silu", "gelu" or "gelu_tanh".
    Any sizes and strides; operands whose rows do not start on 16 bytes are
    copied first.  Differentiable in x, w_in and w_out (once).

    Between the launches a = act(g) u, and for the gradients g, u, dg and du,
    are rounded to x's type.  In float16 such a value past 65504 is infinite and
    one below 6e-5 loses bits, where 32 bits would have held it: the range of
    any float16 network, which losses are scaled for; bfloat16 has that of 32
    bits.
    """
    if not plain_eager(x, w_in, w_out):
        return torch.ops.tensorcore_gemm.gated_ffn(x, w_in, w_out, activation, wants_grad(x, w_in, w_out))[0]
    _check(x, w_in, w_out, activation)
    if wants_grad(x, w_in, w_out):
        return _GatedFfn.apply(x, w_in, w_out, activation)
    return _forward(x, w_in, w_out, activation, False)[0]


# ---------------------------------------------------------------------------
# The dispatcher operators
# ---------------------------------------------------------------------------
@torch.library.custom_op("tensorcore_gemm::gated_ffn", mutates_args=())
def _gated_ffn_op(x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, activation: str,
                  save: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """y and [g u] of `gated_ffn` (the latter is not differentiable; without rows unless `save`d for the gradient)."""
    _check(x, w_in, w_out, activation)
    refuse_tangents(x, w_in, w_out)
    y, gate_up = _forward(x, w_in, w_out, activation, save)
    return y, x.new_empty((0, 2 * _pad8(w_out.shape[1]))) if gate_up is None else gate_up


@_gated_ffn_op.register_fake
def _(x, w_in, w_out, activation, save=True):
    _check(x, w_in, w_out, activation)
    rows = x.shape[:-1].numel() if save else 0
    return (torch.empty((*x.shape[:-1], w_out.shape[0]), dtype=x.dtype, device=x.device),
            torch.empty((rows, 2 * _pad8(w_out.shape[1])), dtype=x.dtype, device=x.device))


@torch.library.custom_op("tensorcore_gemm::gated_ffn_backward", mutates_args=())
def _gated_ffn_backward_op(dy: torch.Tensor, x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor,
                           gate_up: torch.Tensor, activation: str, need_x: bool = True, need_in: bool = True,
                           need_out: bool = True) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """dx, dw_in and dw_out (without elements where not needed)."""
    _check(x, w_in, w_out, activation)
    out_dim, hidden = w_out.shape
    dy = check_operand("dy", dy, (*x.shape[:-1], out_dim), x.dtype, x.device)
    gate_up = check_operand("gate_up", gate_up, (x.shape[:-1].numel(), 2 * _pad8(hidden)), x.dtype, x.device)
    grads = _backward(dy, x, w_in, w_out, gate_up, activation, need_x, need_in, need_out)
    return tuple(x.new_empty(0) if g is None else g for g in grads)


@_gated_ffn_backward_op.register_fake
def _(dy, x, w_in, w_out, gate_up, activation, need_x=True, need_in=True, need_out=True):
    return tuple(torch.empty(t.shape if need else (0,), dtype=t.dtype, device=t.device)
                 for t, need in ((x, need_x), (w_in, need_in), (w_out, need_out)))


def _traced_backward(dy, saved, activation, needs):
    """dx, dw_in and dw_out, those that `needs` names, through the dispatcher; None for the others."""
    grads = torch.ops.tensorcore_gemm.gated_ffn_backward(dy, *saved, activation, *needs[:3])
    return tuple(g if need else None for g, need in zip(grads, needs))


def _setup_context(ctx, inputs, output) -> None:
    x, w_in, w_out, activation, save = inputs
    ctx.save_for_backward(x, w_in, w_out, output[1])
    ctx.activation, ctx.saved = activation, save
    ctx.mark_non_differentiable(output[1])


def _op_backward(ctx, dy, _dgate_up):
    if not ctx.saved:
        raise RuntimeError("gated_ffn was called with save=False: it has no gradient")
    return *_traced_backward(dy, ctx.saved_tensors, ctx.activation, ctx.needs_input_grad), None, None


_gated_ffn_op.register_autograd(_op_backward, setup_context=_setup_context)
