"""The row operators under tracers, dispatch modes and forward mode: traced in full, or refused, never silently wrong."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from tensorcore_gemm import ffn, logprobs, norm


def _norm_args(dev, seed):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x, w, b, dy = (torch.randn(s, generator=gen, device=dev) for s in ((9, 72), (72,), (72,), (9, 72)))
    return (x, w, b), (dy,)


def _ffn_args(dev, seed):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x, wi, wo, dy = (torch.randn(s, generator=gen, device=dev).half() for s in ((9, 64), (80, 64), (24, 40), (9, 24)))
    return (x, wi / 8, wo / 8), (dy,)


def _lprob_args(dev, seed):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x, gl, gh = (torch.randn(s, generator=gen, device=dev) for s in ((9, 300), (9,), (9,)))
    return (x,), (gl, gh)


def _lprob(x):
    r = logprobs.token_logprobs(x, torch.arange(9, device=x.device) * 11, top_k=4)
    return r.logprobs, r.entropy, r.top_logprobs, r.top_indices


# operator -> (call on its differentiable operands, operands and incoming gradients, outputs with a gradient)
OPERATORS = {
    "layer_norm": (lambda x, w, b: (norm.layer_norm(x, w, b),), _norm_args, 1),
    "gated_ffn": (lambda x, wi, wo: (ffn.gated_ffn(x, wi, wo),), _ffn_args, 1),
    "token_logprobs": (_lprob, _lprob_args, 2),
}


def same(a, b):
    return len(a) == len(b) and all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(OPERATORS))
def test_make_fx_on_real_tensors(cuda_device, native_lib, name):
    """A graph recorded from real tensors computes the operator, forward and backward, for other inputs too."""
    call, args, n = OPERATORS[name]
    first, other = args(cuda_device, 1), args(cuda_device, 2)
    graph = make_fx(call, tracing_mode="real")(*first[0])
    assert f"torch.ops.tensorcore_gemm.{name}" in graph.code
    assert same(graph(*other[0]), call(*other[0]))

    def step(leaves, grads):
        leaves = [t.detach().requires_grad_() for t in leaves]
        return torch.autograd.grad(call(*leaves)[:n], leaves, grads)

    graph = make_fx(step, tracing_mode="real")(*first)
    assert same(graph(*other), step(*other))


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(OPERATORS))
def test_backward_under_a_dispatch_mode(cuda_device, native_lib, name):
    """A mode that is entered after the forward sees the backward operator."""
    call, args, n = OPERATORS[name]
    leaves, grads = args(cuda_device, 3)
    leaves = [t.requires_grad_() for t in leaves]
    out = call(*leaves)[:n]
    want = torch.autograd.grad(out, leaves, grads, retain_graph=True)
    seen = []

    class Listen(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    with Listen():
        got = torch.autograd.grad(out, leaves, grads)
    assert same(got, want) and any(f"{name}_backward" in s for s in seen)


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(OPERATORS))
def test_jit_trace(cuda_device, native_lib, name):
    call, args, _ = OPERATORS[name]
    first, other = args(cuda_device, 1)[0], args(cuda_device, 2)[0]
    traced = torch.jit.trace(call, first, check_trace=False)
    assert f"tensorcore_gemm::{name}" in str(traced.graph)
    assert same(traced(*other), call(*other))


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(OPERATORS))
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(cuda_device, native_lib, name, grad):
    """No forward-mode derivative: an operand with a tangent raises, at the entry point and at the dispatcher."""
    call, args, _ = OPERATORS[name]
    operands = args(cuda_device, 1)[0]
    want = call(*operands)
    with forward_ad.dual_level():
        assert same(call(*operands), want)                   # no tangent among them
        for i in range(len(operands)):
            dual = list(operands)
            dual[i] = forward_ad.make_dual(operands[i].clone().requires_grad_(grad), torch.ones_like(operands[i]))
            with pytest.raises(RuntimeError, match="jvp"):
                call(*dual)
        x = forward_ad.make_dual(operands[0].clone().requires_grad_(grad), torch.ones_like(operands[0]))
        rest = {"layer_norm": (*operands[1:], 1e-5), "gated_ffn": (*operands[1:], "silu"),
                "token_logprobs": (torch.arange(9, device=cuda_device), 0, -100)}[name]
        with pytest.raises(RuntimeError, match="jvp"):
            getattr(torch.ops.tensorcore_gemm, name)(x, *rest)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: call(t, *operands[1:])[0], (operands[0],), (torch.ones_like(operands[0]),))


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(OPERATORS))
def test_negated_views(cuda_device, native_lib, name):
    """The imaginary part of a conjugate is a view whose memory holds the negated values."""
    call, args, _ = OPERATORS[name]
    operands = args(cuda_device, 1)[0]
    assert same(call(*(torch._neg_view(t) for t in operands)), call(*(-t for t in operands)))
