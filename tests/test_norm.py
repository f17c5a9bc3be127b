"""Layer norm, forward and backward, against the formulas in 64 bits.

Tolerances.  An output of type T is rounded once: u |y| with u = 2^-11 (fp16),
2^-8 (bf16), 2^-24 (fp32), plus half a subnormal step of fp16.  The fp32
arithmetic behind it sums at most 64 products a thread and then pairwise, so
each sum is off by at most 128 * 2^-24 of the sum of its terms' magnitudes.
The mean's error moves h by rstd * mean|x| of that, called kappa below.
"""
from __future__ import annotations

import pytest
import torch

from tensorcore_gemm import norm

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
TINY = {F16: 2.0 ** -25, BF16: 1e-38, F32: 1e-38}
G = 128 * 2.0 ** -24
EPS = 1e-5


def make(rows, cols, dtype, wdtype, dev, mean=0.5, seed=0):
    gen = torch.Generator().manual_seed(1000 * rows + cols + seed)
    x = torch.randn((rows, cols), generator=gen) + mean * torch.randn((rows, 1), generator=gen)
    w = 1 + 0.1 * torch.randn(cols, generator=gen)
    b = 0.1 * torch.randn(cols, generator=gen)
    dy = torch.randn((rows, cols), generator=gen)
    return x.to(dev, dtype), w.to(dev, wdtype), b.to(dev, wdtype), dy.to(dev, dtype)


def exact(x, w, b, eps=EPS):
    x = x.double()
    mu = x.mean(-1, keepdim=True)
    rstd = (x - mu).square().mean(-1, keepdim=True).add(eps).rsqrt()
    h = (x - mu) * rstd
    w = torch.ones_like(x[0]) if w is None else w.double()
    b = torch.zeros_like(x[0]) if b is None else b.double()
    kappa = 1 + rstd * x.abs().mean(-1, keepdim=True)
    return h, rstd, w, b, kappa


def check_forward(y, x, w, b, eps=EPS):
    h, _, w, b, kappa = exact(x, w, b, eps)
    ref = h * w + b
    bound = UNIT[y.dtype] * ref.abs() + TINY[y.dtype] + G * ((h.abs() + kappa) * w.abs() + b.abs())
    assert y.dtype == x.dtype
    assert ((y.double() - ref).abs() <= bound).all()


def check_backward(dx, dw, db, x, w, dy, eps=EPS):
    h, rstd, w, _, kappa = exact(x, w, None, eps)
    rows, cols = x.shape
    dy = dy.double()
    q = dy * w
    s1, s2 = q.mean(1, keepdim=True), (q * h).mean(1, keepdim=True)
    ref = rstd * (q - s1 - h * s2)
    size = q.abs() + (1 + h.abs()) * (q.abs().mean(1, keepdim=True) + (q * h).abs().mean(1, keepdim=True))
    bound = UNIT[dx.dtype] * ref.abs() + TINY[dx.dtype] + 2 * G * rstd * kappa * size
    assert ((dx.double() - ref).abs() <= bound).all()
    g = (rows + 128) * 2.0 ** -24
    if dw is not None:
        ref = (dy * h).sum(0)
        bound = UNIT[dw.dtype] * ref.abs() + TINY[dw.dtype] + g * (dy.abs() * (h.abs() + kappa)).sum(0)
        assert ((dw.double() - ref).abs() <= bound).all()
    if db is not None:
        ref = dy.sum(0)
        assert ((db.double() - ref).abs() <= UNIT[db.dtype] * ref.abs() + TINY[db.dtype] + g * dy.abs().sum(0)).all()


SIZES = [(1, 1), (1, 8), (5, 7), (3, 64), (33, 257), (600, 256), (2000, 1000), (7, 2048), (1300, 4096), (2, 8192),
         (9, 16384), (700, 520), (3, 9001), (2, 40000), (300, 20008),
         # Several rounds of every block: 16, 32 and 64 columns a thread, one and two rows at once.
         (6001, 2560), (5003, 4096), (4501, 5120), (4003, 1536), (1801, 16384)]
TYPES = [(F16, F16), (F16, F32), (BF16, BF16), (BF16, F32), (F32, F32)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wdtype", TYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_forward_and_gradients(cuda_device, native_lib, rows, cols, dtype, wdtype):
    x, w, b, dy = make(rows, cols, dtype, wdtype, cuda_device)
    check_forward(norm.layer_norm(x, w, b, EPS), x, w, b)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = norm.layer_norm(*leaves, EPS)
    assert torch.equal(y, norm.layer_norm(x, w, b, EPS))
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    check_backward(dx, dw, db, x, w, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("has_w,has_b", [(False, False), (True, False), (False, True)])
def test_without_weight_or_bias(cuda_device, native_lib, has_w, has_b):
    x, w, b, dy = make(70, 384, BF16, F32, cuda_device)
    w, b = (w if has_w else None), (b if has_b else None)
    check_forward(norm.layer_norm(x, w, b), x, w, b)
    leaves = [t.clone().requires_grad_() for t in (x, w, b) if t is not None]
    it = iter(leaves)
    args = [next(it), next(it) if has_w else None, next(it) if has_b else None]
    grads = list(torch.autograd.grad(norm.layer_norm(*args), leaves, dy))
    check_backward(grads[0], grads[1] if has_w else None, grads[-1] if has_b else None, x, w, dy)


@pytest.mark.gpu
def test_only_some_gradients(cuda_device, native_lib):
    x, w, b, dy = make(50, 96, F16, F16, cuda_device)
    w1 = w.clone().requires_grad_()
    dw, = torch.autograd.grad(norm.layer_norm(x, w1, b), (w1,), dy)
    x1 = x.clone().requires_grad_()
    dx, = torch.autograd.grad(norm.layer_norm(x1, w, b), (x1,), dy)
    check_backward(dx, dw, None, x, w, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("offset,pitch,cols", [(0, 200, 136), (1, 201, 136), (8, 264, 136), (3, 150, 133)])
def test_strided_and_misaligned_rows(cuda_device, native_lib, dtype, offset, pitch, cols):
    x0, w, b, dy0 = make(21, pitch, dtype, dtype, cuda_device)
    x, dy = x0[:, offset:offset + cols], dy0[:, offset:offset + cols]
    w, b = w[offset:offset + cols], b[offset:offset + cols]
    check_forward(norm.layer_norm(x, w, b), x, w, b)
    leaf = x0.clone().requires_grad_()
    dx0, = torch.autograd.grad(norm.layer_norm(leaf[:, offset:offset + cols], w, b), (leaf,), dy)
    check_backward(dx0[:, offset:offset + cols], None, None, x, w, dy)
    assert not dx0[:, :offset].any() and not dx0[:, offset + cols:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [257, 4096])
def test_offsets_past_32_bits(cuda_device, native_lib, cols):
    """Rows that start beyond 2^32 elements."""
    rows, pitch = 3, 2 ** 31 + 8
    x0, w, b, dy = make(rows, cols, F16, F32, cuda_device)
    base = torch.empty((rows - 1) * pitch + cols, dtype=F16, device=cuda_device)
    x = base.as_strided((rows, cols), (pitch, 1))
    x.copy_(x0)
    y, stats = norm._forward(x, w, b, EPS, True)
    check_forward(y, x0, w, b)
    dx, dw, db = norm._backward(dy, x, w, stats, F32, True, True)
    check_backward(dx, dw, db, x0, w, dy)


@pytest.mark.gpu
def test_other_layouts(cuda_device, native_lib):
    x, w, b, dy = make(24, 40, F32, F32, cuda_device)
    t = x.t().contiguous().t()                                     # columns contiguous
    check_forward(norm.layer_norm(t, w, b), x, w, b)
    assert torch.equal(norm.layer_norm(x.view(2, 3, 4, 40), w, b).view(24, 40), norm.layer_norm(x, w, b))
    e = x[:1].expand(24, 40)
    check_forward(norm.layer_norm(e, w, b), e, w, b)
    w2 = torch.stack([w, w], 1)[:, 0]                              # strided weight
    assert torch.equal(norm.layer_norm(x, w2, b), norm.layer_norm(x, w, b))
    leaf = x.clone().requires_grad_()
    dx, = torch.autograd.grad(norm.layer_norm(leaf, w, b), (leaf,), dy[:1].expand(24, 40))
    check_backward(dx, None, None, x, w, dy[:1].expand(24, 40))


@pytest.mark.gpu
def test_large_mean_constant_rows_and_bad_rows(cuda_device, native_lib):
    x, w, b, _ = make(40, 1024, F32, F32, cuda_device, mean=300.0)
    check_forward(norm.layer_norm(x, w, b), x, w, b)
    x[3] = 7.25                                                    # no variance: y is the bias
    x[5, 9] = float("nan")
    x[6, 0] = float("inf")
    y = norm.layer_norm(x, w, b)
    assert torch.equal(y[3], b)
    assert y[5].isnan().all() and y[6].isnan().any()
    good = [i for i in range(40) if i not in (3, 5, 6)]
    check_forward(y[good], x[good], w, b)


@pytest.mark.gpu
def test_results_do_not_change_from_run_to_run(cuda_device, native_lib):
    x, w, b, dy = make(5000, 1000, BF16, F32, cuda_device)
    def grads():
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        return torch.autograd.grad(norm.layer_norm(*leaves), leaves, dy)
    first = grads()
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, grads()))


@pytest.mark.gpu
def test_gradient_against_differences(cuda_device, native_lib):
    """<dx, v> against the central difference of sum(dy * y) along v, in 64 bits (step 1e-4: error about 1e-8)."""
    x, w, b, dy = make(6, 50, F32, F32, cuda_device)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(norm.layer_norm(*leaves), leaves, dy)
    gen = torch.Generator().manual_seed(5)
    for i, g in enumerate(grads):
        v = torch.randn(g.shape, generator=gen).to(cuda_device).double()
        def f(s):
            args = [t.double() for t in (x, w, b)]
            args[i] = args[i] + s * v
            h, _, w64, b64, _ = exact(*args)
            return (dy.double() * (h * w64 + b64)).sum()
        diff = (f(1e-4) - f(-1e-4)) / 2e-4
        assert abs((g.double() * v).sum() - diff) <= 1e-5 * (g.double() * v).abs().sum() + 1e-6


@pytest.mark.gpu
def test_empty(cuda_device, native_lib):
    w = torch.ones(16, device=cuda_device, dtype=F16, requires_grad=True)
    x = torch.zeros((0, 16), device=cuda_device, dtype=F16, requires_grad=True)
    y = norm.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == dx.shape == (0, 16) and not dw.any()
    assert norm.layer_norm(torch.zeros((4, 0), device=cuda_device)).shape == (4, 0)


@pytest.mark.gpu
def test_other_stream_and_graph(cuda_device, native_lib):
    x, w, b, _ = make(64, 512, F16, F16, cuda_device)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        big = x.repeat(200, 1)
        y = norm.layer_norm(big, w, b)
    s.synchronize()
    check_forward(y, big, w, b)
    graph = torch.cuda.CUDAGraph()
    buf = x.clone()
    with torch.cuda.graph(graph):
        out = norm.layer_norm(buf, w, b)
    buf.copy_(x * 2)
    graph.replay()
    torch.cuda.synchronize()
    check_forward(out, buf, w, b)


@pytest.mark.gpu
def test_dispatcher_operator(cuda_device, native_lib):
    x, w, b, dy = make(20, 48, F32, F32, cuda_device)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y, stats = torch.ops.tensorcore_gemm.layer_norm(*leaves, EPS)
    assert stats.shape == (2, 20)
    assert torch.equal(y, norm.layer_norm(x, w, b))
    check_backward(*torch.autograd.grad(y, leaves, dy), x, w, dy)
    torch.library.opcheck(torch.ops.tensorcore_gemm.layer_norm, (*leaves, EPS),
                          test_utils=("test_schema", "test_faketensor"))


@pytest.mark.gpu
def test_double_backward_is_refused(cuda_device, native_lib):
    x = torch.randn((4, 16), device=cuda_device, requires_grad=True)
    dx, = torch.autograd.grad(norm.layer_norm(x).square().sum(), (x,), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


@pytest.mark.gpu
def test_refusals(cuda_device, native_lib):
    x = torch.zeros((4, 16), device=cuda_device, dtype=F16)
    ok = torch.zeros(16, device=cuda_device, dtype=F16)
    for bad, match in [((x.double(),), "float16"), ((x, ok[:8]), "1-D"), ((x, ok.bfloat16()), "weight must be"),
                       ((x, ok, ok.float()), "same dtype"), ((x, None, ok.cpu()), "CUDA"),
                       ((x.float(), ok), "weight must be"), ((torch.zeros((), device=cuda_device),), "dimension")]:
        with pytest.raises(RuntimeError, match=match):
            norm.layer_norm(*bad)


def test_cpu_tensors_raise():
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        norm.layer_norm(torch.zeros((4, 16)))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        norm.layer_norm([1.0])


def test_fake_shapes_without_gpu():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode(allow_non_fake_inputs=False):
        x = torch.empty((3, 5, 8), dtype=F16, device="cuda")
        w = torch.empty(8, dtype=F32, device="cuda")
        y = norm.layer_norm(x, w)
        assert y.shape == x.shape and y.dtype == F16
        with pytest.raises(RuntimeError, match="1-D"):
            norm.layer_norm(x, w[:4])


def test_c_argument_checks_without_gpu(native_lib):
    fwd, bwd, size = (native_lib.b200_layer_norm_fwd, native_lib.b200_layer_norm_bwd,
                      native_lib.b200_layer_norm_bwd_workspace_size)
    p = 4096
    assert fwd(p, None, None, p, None, None, -1, 8, 8, 8, 0, 0, EPS, None) == 1
    assert fwd(p, None, None, p, None, None, 4, 8, 8, 8, 7, 7, EPS, None) == 1          # unknown type
    assert fwd(p, None, None, p, None, None, 4, 8, 8, 8, 0, 1, EPS, None) == 1          # fp16 rows, bf16 weight
    assert fwd(p, None, None, p, None, None, 4, 8, 7, 8, 0, 0, EPS, None) == 1          # pitch below the row
    assert fwd(None, None, None, p, None, None, 4, 8, 8, 8, 0, 0, EPS, None) == 1
    assert fwd(p, None, None, p, None, None, 4, 1 << 31, 1 << 31, 1 << 31, 0, 0, EPS, None) == 3
    assert fwd(None, None, None, None, None, None, 0, 8, 8, 8, 0, 0, EPS, None) == 0    # nothing to do
    assert size(-1, 8) == -1 and size(10, 8) == 10 * 2 * 8 * 4
    assert bwd(p, p, None, p, p, p, p, p, 10, 8, 8, 8, 8, 0, 0, p, 639, None) == 8      # workspace one byte short
    assert bwd(p, p, None, p, p, p, p, p, 10, 8, 8, 8, 8, 0, 0, p + 4, 640, None) == 8  # and misaligned


@pytest.mark.gpu
def test_backward_operator_refusals(cuda_device, native_lib):
    """The backward operator refuses what its kernels would read out of range."""
    op = torch.ops.tensorcore_gemm.layer_norm_backward
    x, w, b, dy = make(6, 64, BF16, BF16, cuda_device)
    _, stats = torch.ops.tensorcore_gemm.layer_norm(x, w, b, EPS)
    check_backward(*op(dy, x, w, stats, BF16), x, w, dy)
    check_backward(*op(dy, x, w, stats.t().contiguous().t(), BF16), x, w, dy)
    for args, match in [((dy[:, :32], x, w, stats, BF16), "dy must have shape"), ((dy[:3], x, w, stats, BF16), "dy must have"),
                        ((dy.half(), x, w, stats, BF16), "dy must be"), ((dy.cpu(), x, w, stats, BF16), "CUDA"),
                        ((dy, x, w, stats[:, :3], BF16), "stats must have"), ((dy, x, w, stats.double(), BF16), "stats must be"),
                        ((dy, x, w, stats[:1], BF16), "stats must have"), ((dy, x, w[:8], stats, BF16), "weight must be"),
                        ((dy, x, w, stats, F32), "wdtype"), ((dy, x, None, stats, F16), "wdtype")]:
        with pytest.raises(RuntimeError, match=match):
            op(*args)
