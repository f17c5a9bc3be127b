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


def _compiled(call):
    return torch.compile(call, backend="aot_eager", fullgraph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(OPERATORS))
def test_compiled(cuda_device, native_lib, name):
    call, args, n = OPERATORS[name]
    operands, grads = args(cuda_device, 4)
    assert same(_compiled(call)(*operands), call(*operands))
    results = []
    for f in (_compiled(call), call):
        leaves = [t.clone().requires_grad_() for t in operands]
        results.append(torch.autograd.grad(f(*leaves)[:n], leaves, grads))
    assert same(*results)


class Record(TorchDispatchMode):
    """Shapes of the outputs of the package's operators."""

    def __init__(self):
        super().__init__()
        self.shapes = {}

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if "tensorcore_gemm" in str(func):
            self.shapes[str(func).split(".")[1]] = [tuple(t.shape) for t in out]
        return out


@pytest.mark.gpu
def test_only_what_is_needed_is_computed(cuda_device, native_lib):
    """At the dispatcher, as in eager calls: nothing is kept without a gradient, no gradient of frozen weights."""
    (x, wi, wo), (dy,) = _ffn_args(cuda_device, 5)
    with Record() as seen:
        y = ffn.gated_ffn(x, wi, wo)
    assert seen.shapes == {"gated_ffn": [(9, 24), (0, 80)]}
    for i in range(3):
        operands = [x, wi, wo]
        operands[i] = operands[i].clone().requires_grad_()
        want, = torch.autograd.grad(ffn.gated_ffn(*operands), (operands[i],), dy)
        with Record() as seen:
            z = ffn.gated_ffn(*operands)
            got, = torch.autograd.grad(z, (operands[i],), dy)
        assert torch.equal(z, y) and torch.equal(got, want)
        assert seen.shapes["gated_ffn"] == [(9, 24), (9, 80)]
        assert seen.shapes["gated_ffn_backward"] == [tuple(t.shape) if j == i else (0,) for j, t in enumerate(operands)]
    with pytest.raises(RuntimeError, match="save=False"):
        leaf = x.clone().requires_grad_()
        torch.ops.tensorcore_gemm.gated_ffn(leaf, wi, wo, "silu", False)[0].sum().backward()
    (x, w, b), (dy,) = _norm_args(cuda_device, 5)
    for i in range(3):
        operands = [x, w, b]
        operands[i] = operands[i].clone().requires_grad_()
        want, = torch.autograd.grad(norm.layer_norm(*operands), (operands[i],), dy)
        with Record() as seen:
            got, = torch.autograd.grad(norm.layer_norm(*operands), (operands[i],), dy)
        assert torch.equal(got, want)
        assert seen.shapes["layer_norm_backward"] == [(9, 72), (72,) if i == 1 else (0,), (72,) if i == 2 else (0,)]
