"""The gated feed-forward block, forward and backward, against the formulas in 64 bits.

Tolerances.  Every product sums n 16-bit products in fp32: off by at most
n * 2^-24 of the sum of their magnitudes.  Results, and a, g, u, dg and du
between the launches, are rounded to the operands' type (u = 2^-11 for fp16,
2^-8 for bf16, and half a subnormal step of fp16).  `Exact` carries a bound
beside each value: for a product A B^T with elementwise bounds eA, eB it is
|A| eB + eA |B| + eA eB + n 2^-24 |A||B|, for a function of g the derivative's
maximum times g's bound; approximate exponentials add a relative 2^-19.
"""
from __future__ import annotations

import math

import pytest
import torch

from tensorcore_gemm import _native, ffn

F16, BF16 = torch.float16, torch.bfloat16
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F16: 2.0 ** -25, BF16: 1e-37}
E19 = 2.0 ** -19


def make(rows, dim, hidden, out_dim, dtype, dev, seed=0):
    gen = torch.Generator().manual_seed(rows + 10 * dim + 100 * hidden + seed)
    t = lambda r, c, s: (s * torch.randn((r, c), generator=gen)).to(dtype).to(dev)
    return (t(rows, dim, 1.0), t(2 * hidden, dim, dim ** -0.5), t(out_dim, hidden, hidden ** -0.5),
            t(rows, out_dim, 1.0))


def act64(kind, g):
    """act(g), act'(g), and bounds of |act'| and |act''|."""
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * torch.sigmoid(-g), 1.1, 0.5
    if kind == "gelu":
        c = torch.special.ndtr(g)
        return g * c, c + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi), 1.13, 0.8
    k = math.sqrt(2 / math.pi)
    s = torch.sigmoid(2 * k * (g + 0.044715 * g ** 3))
    return g * s, s + 2 * g * s * (1 - s) * k * (1 + 3 * 0.044715 * g * g), 1.13, 0.85


class Val:
    """A value with an elementwise bound of how far the kernels' may be off."""

    def __init__(self, v, e=None):
        self.v, self.e = v.double(), torch.zeros_like(v, dtype=torch.float64) if e is None else e

    def t(self):
        return Val(self.v.t(), self.e.t())

    def dot(self, b):
        """self @ b^T"""
        a, n = self, self.v.shape[1]
        aa, bb = a.v.abs(), b.v.abs()
        e = aa @ b.e.t() + a.e @ bb.t() + a.e @ b.e.t() + n * 2.0 ** -24 * (aa @ bb.t())
        return Val(a.v @ b.v.t(), e)

    def times(self, b):
        e = self.v.abs() * b.e + self.e * b.v.abs() + self.e * b.e
        v = self.v * b.v
        return Val(v, e + 2.0 ** -23 * v.abs())

    def rounded(self, dtype):
        return Val(self.v, self.e + UNIT[dtype] * (self.v.abs() + self.e) + TINY[dtype])

    def check(self, got):
        assert ((got.double() - self.v).abs() <= self.e).all(), ((got.double() - self.v).abs() / self.e).max()


class Exact:
    def __init__(self, x, w_in, w_out, kind, dy=None):
        dt = x.dtype
        hidden = w_out.shape[1]
        X, Wi, Wo = Val(x), Val(w_in), Val(w_out)
        gu = X.dot(Wi)
        g, u = Val(gu.v[:, :hidden], gu.e[:, :hidden]), Val(gu.v[:, hidden:], gu.e[:, hidden:])

        def apply(g):
            f, s, l1, l2 = act64(kind, g.v)
            fe = l1 * g.e + E19 * (f.abs() + 2.0 ** -4 * g.v.abs())
            return Val(f, fe), Val(s, l2 * g.e + E19 * (1 + g.v.abs()))

        self.y = apply(g)[0].times(u).rounded(dt).dot(Wo).rounded(dt)
        if dy is None:
            return
        DY = Val(dy)
        g, u = g.rounded(dt), u.rounded(dt)
        f, s = apply(g)
        a = f.times(u).rounded(dt)
        da = DY.dot(Wo.t())
        dg, du = da.times(u).times(s).rounded(dt), da.times(f).rounded(dt)
        dgu = Val(torch.cat([dg.v, du.v], 1), torch.cat([dg.e, du.e], 1))
        self.dx = dgu.dot(Wi.t()).rounded(dt)
        self.dw_in = dgu.t().dot(X.t()).rounded(dt)
        self.dw_out = DY.t().dot(a.t()).rounded(dt)


def run(x, w_in, w_out, kind, dy):
    leaves = [t.detach().clone().requires_grad_() for t in (x, w_in, w_out)]
    y = ffn.gated_ffn(*leaves, activation=kind)
    return y, *torch.autograd.grad(y, leaves, dy)


def check_all(x, w_in, w_out, kind, dy):
    ex = Exact(x, w_in, w_out, kind, dy)
    y, dx, dwi, dwo = run(x, w_in, w_out, kind, dy)
    ex.y.check(ffn.gated_ffn(x, w_in, w_out, activation=kind))
    for want, got, like in ((ex.y, y, dy), (ex.dx, dx, x), (ex.dw_in, dwi, w_in), (ex.dw_out, dwo, w_out)):
        assert got.shape == like.shape and got.dtype == like.dtype
        want.check(got)


# rows, dim, hidden, out_dim: one row, few, odd ones, sizes around the tiles (256 rows, 128 hidden units, 64 deep)
SIZES = [(1, 8, 8, 8), (1, 256, 512, 256), (3, 64, 128, 64), (17, 100, 60, 100), (33, 129, 131, 65),
         (128, 128, 128, 128),
         (130, 200, 264, 200), (256, 512, 1000, 512), (257, 511, 1001, 510), (700, 96, 384, 104), (1500, 320, 72, 320),
         (64, 1024, 2816, 1024), (2, 2000, 33, 7), (520, 384, 776, 392), (1111, 130, 267, 131), (300, 2048, 136, 72),
         (2600, 64, 200, 264)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(ffn.ACTIVATIONS))
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("size", SIZES)
def test_forward_and_gradients(cuda_device, native_lib, size, dtype, kind):
    x, w_in, w_out, dy = make(*size, dtype, cuda_device)
    check_all(x, w_in, w_out, kind, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [2, 5, 8, 9, 15, 16, 24, 31, 32, 48, 63, 65, 100, 127, 129, 200, 255, 300])
def test_row_counts(cuda_device, native_lib, rows, dtype):
    """Every row count near where the kernels change."""
    x, w_in, w_out, _ = make(rows, 384, 776, 392, dtype, cuda_device)
    Exact(x, w_in, w_out, "silu").y.check(ffn.gated_ffn(x, w_in, w_out))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 20, 300])
def test_large_gates(cuda_device, native_lib, rows):
    """Gates far into both tails: no overflow on the way."""
    x, w_in, w_out, dy = make(rows, 64, 136, 64, BF16, cuda_device)
    w_in = w_in.clone()
    w_in[:136] *= 100
    for kind in ffn.ACTIVATIONS:
        y, dx, dwi, dwo = run(x, w_in, w_out, kind, dy)
        ex = Exact(x, w_in, w_out, kind)
        ex.y.check(y)
        assert all(t.isfinite().all() for t in (y, dx, dwi, dwo))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_strided_operands(cuda_device, native_lib, rows):
    x, w_in, w_out, dy = make(rows, 200, 160, 120, F16, cuda_device)
    want = Exact(x[:, 8:136], w_in[:, 16:144], w_out[:, :160], "silu", dy[:, :120])
    y, dx, dwi, dwo = run(x[:, 8:136], w_in[:, 16:144], w_out[:, :160], "silu", dy[:, :120])
    want.y.check(y)
    leaf = [t.clone().requires_grad_() for t in (x, w_in, w_out)]
    y = ffn.gated_ffn(leaf[0][:, 8:136], leaf[1][:, 16:144], leaf[2])
    want.y.check(y)
    g = torch.autograd.grad(y, leaf, dy)
    want.dx.check(g[0][:, 8:136])
    want.dw_in.check(g[1][:, 16:144])
    want.dw_out.check(g[2])
    # misaligned columns, transposed storage, expanded rows, more dimensions
    Exact(x[:, 3:131], w_in[:, 1:129], w_out, "gelu").y.check(
        ffn.gated_ffn(x[:, 3:131], w_in[:, 1:129], w_out, activation="gelu"))
    xt, wit, wot = (t.t().contiguous().t() for t in (x, w_in, w_out))
    Exact(x, w_in, w_out, "silu").y.check(ffn.gated_ffn(xt, wit, wot))
    e = x[:1].expand(rows, 200)
    Exact(e, w_in, w_out, "silu").y.check(ffn.gated_ffn(e, w_in, w_out))
    assert torch.equal(ffn.gated_ffn(x.view(rows, 1, 200), w_in, w_out).view(rows, 120), ffn.gated_ffn(x, w_in, w_out))


@pytest.mark.gpu
@pytest.mark.parametrize("pitch", [2 ** 31 + 8, 2 ** 31 + 1])
def test_offsets_past_32_bits(cuda_device, native_lib, pitch):
    """Rows of x that start beyond 2^32 elements, aligned or not."""
    x0, w_in, w_out, _ = make(3, 72, 40, 24, F16, cuda_device)
    base = torch.empty(2 * pitch + 72, dtype=F16, device=cuda_device)
    x = base.as_strided((3, 72), (pitch, 1))
    x.copy_(x0)
    Exact(x0, w_in, w_out, "silu").y.check(ffn.gated_ffn(x, w_in, w_out))


@pytest.mark.gpu
def test_only_some_gradients(cuda_device, native_lib):
    x, w_in, w_out, dy = make(70, 64, 96, 80, BF16, cuda_device)
    full = run(x, w_in, w_out, "silu", dy)[1:]
    for i in range(3):
        args = [x, w_in, w_out]
        args[i] = args[i].clone().requires_grad_()
        g, = torch.autograd.grad(ffn.gated_ffn(*args), (args[i],), dy)
        assert torch.equal(g, full[i])


@pytest.mark.gpu
def test_nan_stays_in_its_row(cuda_device, native_lib):
    for rows in (6, 300):
        x, w_in, w_out, _ = make(rows, 128, 256, 128, F16, cuda_device)
        x = x.clone()
        x[2, 5] = float("nan")
        y = ffn.gated_ffn(x, w_in, w_out)
        assert y[2].isnan().all()
        good = [i for i in range(rows) if i != 2]
        Exact(x[good], w_in, w_out, "silu").y.check(y[good])


@pytest.mark.gpu
def test_results_do_not_change_from_run_to_run(cuda_device, native_lib):
    for rows in (4, 40, 900):
        x, w_in, w_out, dy = make(rows, 512, 1400, 512, BF16, cuda_device)
        first = run(x, w_in, w_out, "silu", dy)
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(first, run(x, w_in, w_out, "silu", dy)))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(ffn.ACTIVATIONS))
def test_gradient_against_differences(cuda_device, native_lib, kind):
    """The gradient along v against the central difference of the 64-bit function (step 1e-4, error about 1e-7).

    The kernels' gradient of 64 x 48 elements carries roundings of 2^-11 that are independent of v, each
    weighted with at most its value; four standard deviations of their sum are allowed."""
    x, w_in, w_out, dy = make(64, 48, 56, 48, F16, cuda_device)
    grads = run(x, w_in, w_out, kind, dy)[1:]
    gen = torch.Generator().manual_seed(2)
    for i, g in enumerate(grads):
        v = torch.randn(g.shape, generator=gen).to(cuda_device).double()

        def f(s):
            args = [t.double() for t in (x, w_in, w_out)]
            args[i] = args[i] + s * v
            gate, up = (args[0] @ args[1].t()).chunk(2, 1)
            return (dy.double() * ((act64(kind, gate)[0] * up) @ args[2].t())).sum()

        diff = (f(1e-4) - f(-1e-4)) / 2e-4
        got = (g.double() * v).sum()
        # roundings on the way: of g, u (through a smooth function), a or dg and du, and the result
        assert abs(got - diff) <= 4 * 4 * 2.0 ** -11 * (g.double() * v).square().sum().sqrt() + 1e-4


@pytest.mark.gpu
def test_empty(cuda_device, native_lib):
    for rows, dim, hidden, out_dim in [(0, 16, 8, 16), (5, 0, 8, 16), (5, 16, 0, 16), (5, 16, 8, 0)]:
        x, w_in, w_out, dy = (torch.ones(s, device=cuda_device, dtype=F16) for s in
                              ((rows, dim), (2 * hidden, dim), (out_dim, hidden), (rows, out_dim)))
        for t in run(x, w_in, w_out, "silu", dy):
            assert not t.any()
        assert not ffn.gated_ffn(x, w_in, w_out).any()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 30, 400])
def test_stream_and_graph(cuda_device, native_lib, rows):
    x, w_in, w_out, _ = make(rows, 512, 1024, 512, F16, cuda_device)
    ex = Exact(x, w_in, w_out, "silu")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(20):                              # back to back, weights written just before their use
            wi, wo = w_in * 1.0, w_out * 1.0
            y = ffn.gated_ffn(x, wi, wo)
    s.synchronize()
    ex.y.check(y)
    buf = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ffn.gated_ffn(buf, w_in, w_out)
    buf.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    ex.y.check(out)


@pytest.mark.gpu
def test_dispatcher_operator(cuda_device, native_lib):
    x, w_in, w_out, dy = make(40, 64, 72, 64, F16, cuda_device)
    leaves = [t.clone().requires_grad_() for t in (x, w_in, w_out)]
    y, gate_up = torch.ops.tensorcore_gemm.gated_ffn(*leaves, "silu")
    assert gate_up.shape == (40, 144)
    for p, q in zip((y, *torch.autograd.grad(y, leaves, dy)), run(x, w_in, w_out, "silu", dy)):
        assert torch.equal(p, q)
    torch.library.opcheck(torch.ops.tensorcore_gemm.gated_ffn, (*leaves, "silu"),
                          test_utils=("test_schema", "test_faketensor"))


@pytest.mark.gpu
def test_refusals(cuda_device, native_lib):
    x, w_in, w_out, _ = make(4, 16, 8, 16, F16, cuda_device)
    for args, match in [((x.float(), w_in, w_out), "float16 or bfloat16"), ((x, w_in.bfloat16(), w_out), "dtype"),
                        ((x, w_in[:, :8], w_out), "Inner"), ((x, w_in[:15], w_out), "twice"),
                        ((x, w_in, w_out.cpu()), "CUDA"), ((x, w_in[0], w_out), "two")]:
        with pytest.raises(RuntimeError, match=match):
            ffn.gated_ffn(*args)
    with pytest.raises(ValueError, match="Unsupported activation"):
        ffn.gated_ffn(x, w_in, w_out, activation="relu")
    a = x.clone().requires_grad_()
    dx, = torch.autograd.grad(ffn.gated_ffn(a, w_in, w_out).sum(), (a,), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


def test_cpu_tensors_raise():
    t = torch.zeros((8, 8), dtype=F16)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ffn.gated_ffn(t, torch.zeros((16, 8), dtype=F16), t)


def test_fake_shapes_without_gpu():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode(allow_non_fake_inputs=False):
        x = torch.empty((3, 5, 16), dtype=BF16, device="cuda")
        w_in, w_out = (torch.empty(s, dtype=BF16, device="cuda") for s in ((22, 16), (24, 11)))
        y = ffn.gated_ffn(x, w_in, w_out)
        assert y.shape == (3, 5, 24) and y.dtype == BF16
        with pytest.raises(RuntimeError, match="twice"):
            ffn.gated_ffn(x, w_in[:20], w_out)


def test_c_argument_checks_without_gpu(native_lib):
    size, fwd, bwd = (native_lib.b200_gated_ffn_workspace_size, native_lib.b200_gated_ffn_fwd,
                      native_lib.b200_gated_ffn_bwd)
    p = 4096
    assert size(-1, 8, 8, 8, 0, 0) == -1 and size(4, 64, 64, 64, 0, 0) == 512 and size(4, 64, 64, 64, 1, 0) == 1536
    assert size(4, 64, 64, 1 << 31, 0, 0) == -3 and size(4, 64, 60, 64, 0, 0) > 512 and size(4, 64, 64, 64, 0, 1) > 512
    args = [p] * 5 + [4, 64, 64, 64, 64, 64, 64, 64, 0, 1, p, 1 << 20, None]
    def with_(a, i, v):
        return [v if j == i else q for j, q in enumerate(a)]
    for i, v, code in [(0, None, 1), (1, None, 1), (2, None, 1), (3, None, 1), (5, -1, 1), (5, 1 << 31, 3), (7, -1, 1),
                       (9, 63, 1), (12, 60, 1), (13, 3, 1), (14, 2, 1), (15, None, 8), (15, p + 8, 8),
                       (16, 511, 8), (4, p + 2, 2)]:
        assert fwd(*with_(args, i, v)) == code, (i, v)
    args = [p] * 8 + [4, 64, 64, 64] + [64] * 7 + [0, 1, p, 1 << 20, None]
    for i, v, code in [(0, None, 1), (4, None, 1), (4, p + 2, 2), (16, 63, 1), (18, 60, 1),
                       (21, p + 8, 8), (22, 1535, 8)]:
        assert bwd(*with_(args, i, v)) == code, (i, v)


# The products of a pass of (rows, dim, hidden, out_dim) as b200_gated_ffn_plan takes them.
def products(rows, dim, hidden, out_dim):
    pad = -(-hidden // 8) * 8
    return {"gate_up": (rows, hidden, dim), "out": (rows, out_dim, hidden), "gate_grad": (rows, hidden, out_dim),
            "in_grad": (rows, dim, 2 * pad)}


SM_SHARED, CTA_RESERVED, TMEM_COLUMNS = 228 * 1024, 1024, 512   # of an SM; of each CTA; of an SM


def test_few_rows_ctas_never_wait_for_tensor_memory(native_lib):
    """CTAs of the few-rows kernel that share an SM find tensor memory for all of them.

    A CTA whose allocation waited would hold up its cluster, and clusters that each hold what another one's CTA
    waits for would never end.  With its share of the SM's shared memory at least its share of the tensor memory,
    CTAs that fit the one fit the other, whichever launches they come from."""
    seen = set()
    for rows in (1, 8, 16, 17, 33, 64, 65, 100, 128, 129, 200, 256, 257, 400, 512, 700, 1500, 4000):
        for n in (8, 64, 72, 128, 200, 384, 512, 1000, 2048, 2731, 4096, 12288):
            for k in (8, 64, 128, 192, 256, 320, 512, 520, 1024, 2048, 4096, 12288):
                for product in _native.FFN_PRODUCTS:
                    ctas, smem, columns = _native.gated_ffn_plan(rows, n, k, product)
                    if ctas:
                        seen.add((ctas, columns))
                        assert (smem + CTA_RESERVED) * TMEM_COLUMNS >= columns * SM_SHARED, (rows, n, k, product)
                        assert smem <= SM_SHARED - CTA_RESERVED
    assert {c for c, _ in seen} == {1, 2, 4, 8} and {t for _, t in seen} == {32, 64, 128, 256, 512}


@pytest.mark.gpu
def test_backward_operator_refusals(cuda_device, native_lib):
    """The backward operator refuses what its kernels would read out of range."""
    op = torch.ops.tensorcore_gemm.gated_ffn_backward
    x, w_in, w_out, dy = make(40, 64, 70, 56, F16, cuda_device)
    _, gu = torch.ops.tensorcore_gemm.gated_ffn(x, w_in, w_out, "silu")
    for p, q in zip(op(dy, x, w_in, w_out, gu, "silu"), run(x, w_in, w_out, "silu", dy)[1:]):
        assert torch.equal(p, q)
    assert torch.equal(op(dy, x, w_in, w_out, gu.t().contiguous().t(), "silu")[0], op(dy, x, w_in, w_out, gu, "silu")[0])
    for args, match in [((dy[:, :40], x, w_in, w_out, gu), "dy must have shape"), ((dy[:8], x, w_in, w_out, gu), "dy must have"),
                        ((dy.float(), x, w_in, w_out, gu), "dy must be"), ((dy.cpu(), x, w_in, w_out, gu), "CUDA"),
                        ((dy, x, w_in, w_out, gu[:8]), "gate_up must have"), ((dy, x, w_in, w_out, gu[:, :140]), "gate_up must"),
                        ((dy, x, w_in, w_out, gu.bfloat16()), "gate_up must be"), ((dy, x, w_in[:, :32], w_out, gu), "Inner"),
                        ((dy, x[:8], w_in, w_out, gu), "dy must have")]:
        with pytest.raises(RuntimeError, match=match):
            op(*args, "silu")
    with pytest.raises(ValueError, match="Unsupported activation"):
        op(dy, x, w_in, w_out, gu, "relu")


def test_dimension_limits_without_gpu(native_lib):
    """Sizes whose rounding up would pass 32 bits are refused, not wrapped (2 hidden as a depth, above all)."""
    size, fwd, bwd = (native_lib.b200_gated_ffn_workspace_size, native_lib.b200_gated_ffn_fwd,
                      native_lib.b200_gated_ffn_bwd)
    p, most = 4096, 0x7f000000
    for dims in [(1, 8, 0x3fffffff, 8), (1, 8, most // 2 + 1, 8), (most + 1, 8, 8, 8), (0x7fffffff, 1, 1, 1),
                 (1, most + 1, 8, 8), (1, 8, 8, 0x7fffffff)]:
        rows, dim, hidden, out_dim = dims
        assert size(*dims, 0, 0) == size(*dims, 1, 0) == -3
        assert fwd(*[p] * 5, *dims, dim, dim, hidden, out_dim, 0, 1, p, 1 << 62, None) == 3
        assert bwd(*[p] * 8, *dims, out_dim, dim, dim, hidden, dim, dim, hidden, 0, 1, p, 1 << 62, None) == 3
    assert size(1, 8, most // 2, 8, 1, 0) > 0 and size(1, most, 8, 8, 1, 0) > 0 and size(most, 8, 8, 8, 1, 0) > 0
    for product in _native.FFN_PRODUCTS:                    # the plan's own arithmetic at the limits
        for rows, n, k in [(1, most, 8), (300, most, 64), (1, 8, most), (most, 8, 8)]:
            ctas, smem, columns = _native.gated_ffn_plan(rows, n, k, product)
            assert ctas in (0, 1, 2, 4, 8) and 0 <= smem <= 227 * 1024 and columns <= 512


# A training step whose dw_out is a product that the GEMM splits along K in its last wave.
SPLIT = (8192, 64, 2048, 2560)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_split_products_use_the_callers_workspace(cuda_device, native_lib, dtype):
    """No device memory is allocated, whatever the stream, and a captured step computes what an eager one does."""
    rows, dim, hidden, out_dim = SPLIT
    assert _native.plan(out_dim, hidden, rows) == ("pair", 4)
    x, w_in, w_out, dy = make(*SPLIT, dtype, cuda_device)
    check_all(x, w_in, w_out, "silu", dy)
    code = 0 if dtype == F16 else 1
    gu = torch.empty((rows, 2 * hidden), dtype=dtype, device=cuda_device)
    y, dx, dwi, dwo = (torch.empty_like(t) for t in (dy, x, w_in, w_out))
    ws = torch.empty(native_lib.b200_gated_ffn_workspace_size(*SPLIT, 1, 0), dtype=torch.uint8, device=cuda_device)

    def step(stream):
        p = [t.data_ptr() for t in (x, w_in, w_out, y, gu)]
        assert native_lib.b200_gated_ffn_fwd(*p, *SPLIT, dim, dim, hidden, out_dim, 0, code, ws.data_ptr(), ws.numel(),
                                             stream.cuda_stream) == 0
        p = [t.data_ptr() for t in (dy, x, w_in, w_out, gu, dx, dwi, dwo)]
        assert native_lib.b200_gated_ffn_bwd(*p, *SPLIT, out_dim, dim, dim, hidden, dim, dim, hidden, 0, code,
                                             ws.data_ptr(), ws.numel(), stream.cuda_stream) == 0

    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    step(streams[0])
    streams[0].synchronize()
    want = [t.clone() for t in (y, dx, dwi, dwo)]
    free = torch.cuda.mem_get_info()[0]
    ws.fill_(255)                                            # leftovers of another use
    torch.cuda.synchronize()
    step(streams[1])
    streams[1].synchronize()
    assert torch.cuda.mem_get_info()[0] == free
    assert all(torch.equal(p, q) for p, q in zip((y, dx, dwi, dwo), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream())
    for t in (y, dx, dwi, dwo):
        t.zero_()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip((y, dx, dwi, dwo), want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_variant_override_leaves_the_block_alone(cuda_device, native_lib, dtype):
    """b200_gemm_set_variant steers the GEMM's entry points; the block chooses for itself, in both types alike."""
    x, w_in, w_out, dy = make(*SPLIT, dtype, cuda_device)
    want = run(x, w_in, w_out, "silu", dy)
    try:
        for variant in ("cta1", "pair", "pair2m"):
            _native.set_variant(variant)
            assert all(torch.equal(p, q) for p, q in zip(run(x, w_in, w_out, "silu", dy), want))
    finally:
        _native.set_variant("auto")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40, 300, 4100])
@pytest.mark.parametrize("kind", list(ffn.ACTIVATIONS))
def test_gates_whose_square_overflows(cuda_device, native_lib, kind, rows):
    """bf16 gates of +-1e20: the slope is 1 or 0, whatever g^2 is."""
    x, w_in, w_out, dy = make(rows, 64, 72, 64, BF16, cuda_device)
    x, w_in = x.clone(), w_in.clone()
    x[:, 0] = 1.0
    w_in[3, 0], w_in[70, 0] = 1e20, -1e20
    ex = Exact(x, w_in, w_out, kind, dy)
    for want, got in zip((ex.y, ex.dx, ex.dw_in, ex.dw_out), run(x, w_in, w_out, kind, dy)):
        assert got.isfinite().all()
        want.check(got)


# Every product on the GEMM's tiles (256 rows; 128 columns of gate and up, 256 of da; 128 deep): less than a tile and
# several in each direction, hidden widths off 8, one stage of depth and several, more tiles than pairs of SMs.
MANY_ROWS = [(4097, 8, 8, 8), (4100, 64, 267, 72), (4353, 200, 1000, 136), (4609, 520, 2731, 264), (5000, 136, 135, 640)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(ffn.ACTIVATIONS))
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("size", MANY_ROWS)
def test_many_rows(cuda_device, native_lib, size, dtype, kind):
    """The epilogues of the pair kernel, forward and backward, and the GEMMs beside them."""
    for product, args in products(*size).items():
        assert _native.gated_ffn_plan(*args, product) == (0, 0, 0), product
    x, w_in, w_out, dy = make(*size, dtype, cuda_device)
    check_all(x, w_in, w_out, kind, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(ffn.ACTIVATIONS))
def test_many_rows_strided_and_repeated(cuda_device, native_lib, kind):
    """Operands with pitches and off 16 bytes, a NaN row, the same bits from run to run."""
    rows, dim, hidden, out_dim = 4201, 136, 530, 200
    x, w_in, w_out, dy = make(rows, dim + 8, hidden, out_dim + 8, BF16, cuda_device)
    for a, b in ((8, 8), (3, 1)):
        xs, wi, wo, dys = x[:, a:a + dim], w_in[:, b:b + dim], w_out[b:b + out_dim], dy[:, a:a + out_dim]
        ex = Exact(xs, wi, wo, kind, dys)
        leaves = [t.detach().requires_grad_() for t in (xs, wi, wo)]
        y = ffn.gated_ffn(*leaves, activation=kind)
        first = (y, *torch.autograd.grad(y, leaves, dys))
        for want, got in zip((ex.y, ex.dx, ex.dw_in, ex.dw_out), first):
            want.check(got)
        y = ffn.gated_ffn(*leaves, activation=kind)
        assert all(torch.equal(p, q) for p, q in zip(first, (y, *torch.autograd.grad(y, leaves, dys))))
    bad = xs.clone()
    bad[7, 5] = float("nan")
    y = ffn.gated_ffn(bad, wi, wo, activation=kind)
    assert y[7].isnan().all() and torch.equal(torch.cat([y[:7], y[8:]]), torch.cat([first[0][:7], first[0][8:]]))


# Sizes whose products run on each kernel of the GEMM, with the product and the kernel that it is there for.
KERNELS = [((4100, 2008, 520, 2008), {"out": "pair2m", "in_grad": "pair2m"}),
           ((5000, 1000, 520, 1000), {"out": "pair2m_192", "in_grad": "pair2m_192"}),
           ((5000, 1500, 520, 1500), {"out": "pair2m_224", "in_grad": "pair2m_224"}),
           ((4100, 520, 520, 2600), {"out": "pair", "in_grad": "cta1", "dw_in": "pair", "dw_out": "pair"}),
           ((5000, 2008, 520, 520), {"out": "cta1", "in_grad": "pair"}),
           ((4100, 1500, 2600, 520), {"dw_in": "pair2m"}), ((4100, 2600, 1500, 520), {"dw_in": "pair2m_224"}),
           ((4100, 520, 2600, 2600), {"dw_out": "pair2m_224"}), ((4100, 520, 3500, 2600), {"dw_out": "cta1"})]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("size,kernels", KERNELS)
def test_every_gemm_kernel(cuda_device, native_lib, size, kernels, dtype):
    """The wide pair in its three widths, the pair and the one-CTA kernel behind the block, in both types."""
    rows, dim, hidden, out_dim = size
    args = dict(products(*size), dw_in=(2 * hidden, dim, rows), dw_out=(out_dim, hidden, rows))
    for product, kernel in kernels.items():
        assert _native.plan(*args[product])[0] == kernel
        if product in _native.FFN_PRODUCTS:
            assert _native.gated_ffn_plan(*args[product], product) == (0, 0, 0)
    x, w_in, w_out, dy = make(*size, dtype, cuda_device)
    check_all(x, w_in, w_out, "silu", dy)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 300, 4100])
def test_range_between_the_launches(cuda_device, native_lib, rows):
    """a, dg and du past fp16's range are infinite in fp16, in their rows only; bf16 holds them."""
    for dtype in (F16, BF16):
        x, w_in, w_out, dy = make(rows, 64, 72, 64, dtype, cuda_device)
        x, w_in, dy = x.clone(), w_in.clone(), dy.clone()
        w_in[5] = w_in[77] = 0.0
        w_in[5, 0] = w_in[77, 0] = 1.0                       # g and u of unit 5
        x[1, 0] = 400.0                                      # a = 160000
        x[2, 0], dy[2] = 200.0, 4000.0 * w_out[:, 5].sign()  # a = 40000, dg = da u far past the range
        y, dx, dwi, dwo = run(x, w_in, w_out, "silu", dy)
        rest = [i for i in range(rows) if i not in (1, 2)]
        if rest:
            ex = Exact(x[rest], w_in, w_out, "silu", dy[rest])
            ex.y.check(y[rest])
            ex.dx.check(dx[rest])
        if dtype == F16:
            assert not y[1].isfinite().any() and not dx[2].isfinite().all() and not dwo.isfinite().all()
        else:
            ex = Exact(x, w_in, w_out, "silu", dy)
            for want, got in ((ex.y, y), (ex.dx, dx), (ex.dw_in, dwi), (ex.dw_out, dwo)):
                assert got.isfinite().all()
                want.check(got)
