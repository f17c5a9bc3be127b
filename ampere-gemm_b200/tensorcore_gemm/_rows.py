"""Helpers of the operators that work on the rows of a tensor (norm, ffn,
logprobs): argument checks, the 2-D view the C ABI takes, workspaces and the
launch on torch's current stream."""
from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad

from . import _native
from .gemm import _GET_DEVICE, _current_stream

DTYPE_CODES = {
    torch.float16: _native.B200_DTYPE_F16,
    torch.bfloat16: _native.B200_DTYPE_BF16,
    torch.float32: _native.B200_DTYPE_F32,
}


def check_cuda(name: str, t, dtypes=tuple(DTYPE_CODES)) -> None:
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if t.dtype not in dtypes:
        raise RuntimeError(f"{name} must be {' or '.join(str(d).replace('torch.', '') for d in dtypes)}")


def check_operand(name: str, t, shape, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """`t`, contiguous, or an error where it is not what the kernels will read it as."""
    check_cuda(name, t, (dtype,))
    if t.shape != torch.Size(shape):
        raise RuntimeError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    if t.device != device:
        raise RuntimeError(f"{name} must be on {device}")
    return t.contiguous()


def as_rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """`t` as a matrix of its last dimension's rows, and its row pitch.

    A row-strided view (a column slice) is used in place; anything else, an
    expanded tensor among them, is made contiguous."""
    if t.dim() != 2:
        cols = t.shape[-1]
        t = t.reshape(-1, cols) if cols else t.reshape(0, 0)
    rows, cols = t.shape
    if cols <= 1:
        cols = 1
        if rows <= 1 or t.stride(0) >= 1:
            return t, cols if rows <= 1 else t.stride(0)
    else:
        pitch, unit = t.stride()
        if unit == 1:
            if rows <= 1:
                return t, cols
            if pitch >= cols:
                return t, pitch
    return t.contiguous(), cols


def workspace(nbytes: int, device: torch.device, what: str) -> torch.Tensor | None:
    """Device memory for a call (None when it needs none); freed to torch's
    allocator, which reuses it in stream order."""
    if nbytes < 0:
        _native.check(-nbytes, what)
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


_FUNCTIONS: dict = {}


def launch(name: str, dev: int, *args) -> None:
    """Calls C entry point `name` with `args` and the current stream of device `dev`; raises on an error code."""
    fn = _FUNCTIONS.get(name)
    if fn is None:
        fn = _FUNCTIONS[name] = getattr(_native.load(), name)
    if dev != _GET_DEVICE():
        with torch.cuda.device(dev):
            code = fn(*args, _current_stream(dev))
    else:
        code = fn(*args, _current_stream(dev))
    if code != _native.B200_OK:
        _native.check(code, name)


_DISPATCH_MODES, _JIT_TRACE = torch._C._len_torch_dispatch_stack, torch._C._get_tracing_state


def plain_eager(*tensors) -> bool:
    """True when the call can go straight to the kernels: real tensors, and nobody who listens at the dispatcher
    (a compiler, a dispatch mode such as make_fx's, torch.jit.trace) or works through it (negated views)."""
    if torch.compiler.is_compiling() or _DISPATCH_MODES() or _JIT_TRACE() is not None:
        return False
    for t in tensors:
        if isinstance(t, torch.Tensor) and (type(t) not in (torch.Tensor, torch.nn.Parameter) or t.is_neg()):
            return False
    return True


def wants_grad(*tensors) -> bool:
    """True when the call has to be an autograd.Function's: gradients are wanted, or, within a dual level, may be
    (the Function raises for an operand with a tangent, as it has no forward-mode derivative)."""
    if forward_ad._current_level >= 0:
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def refuse_tangents(*tensors) -> None:
    """For the dispatcher operators, which torch.library would otherwise let drop a tangent."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("this operator has no forward-mode derivative (jvp)")


class _Refuse(torch.autograd.Function):
    """Identity whose differentiation raises."""

    @staticmethod
    def forward(ctx, *tensors):
        return tuple(t.view_as(t) for t in tensors)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("this gradient cannot be differentiated again: the operator is once_differentiable")


def once_differentiable(backward):
    """A Function's backward whose results refuse to be differentiated.

    torch's decorator of that name lets a second differentiation through,
    as a constant, when the incoming gradient needs none itself."""

    @functools.wraps(backward)
    def wrapper(ctx, *grads):
        if not torch.is_grad_enabled():          # the usual case: no create_graph=True
            return backward(ctx, *grads)
        with torch.no_grad():
            out = backward(ctx, *grads)
        at = [i for i, t in enumerate(out) if t is not None]
        refused = _Refuse.apply(*(out[i].detach().requires_grad_() for i in at)) if at else ()
        out = list(out)
        for i, t in zip(at, refused):
            out[i] = t
        return tuple(out)

    return wrapper
