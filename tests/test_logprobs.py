"""Token log probabilities, entropies, top alternatives and the logits' gradient against the formulas in 64 bits.

Tolerances.  With d = x - max, an fp32 exp(d) is off by a relative 2^-22 (the
approximate power of two) and by 2^-23 |d| (the rounded exponent); sums over a
thread's logits and then pairwise add less than 2^-20 of the (positive) sum.
So ln z is off by at most 2^-20 + 2^-22 E|d| (E: the mean under the softmax),
which logprob has beside its own rounding, the entropy's second term by as much
times E|d| and by E d^2 of it, and a gradient element by that share of its terms.
A gradient is rounded once to the logits' type (u as below).
"""
from __future__ import annotations

import math

import pytest
import torch

from tensorcore_gemm import logprobs

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
TINY = {F16: 2.0 ** -25, BF16: 1e-37, F32: 1e-37}
E20, E22 = 2.0 ** -20, 2.0 ** -22


def make(rows, vocab, dtype, dev, std=3.0, barred=0.0, seed=0):
    gen = torch.Generator().manual_seed(7 * rows + vocab + seed)
    x = (std * torch.randn((rows, vocab), generator=gen)).to(dtype)
    if barred:
        x[torch.rand(x.shape, generator=gen) < barred] = -math.inf
    t = torch.randint(0, vocab, (rows,), generator=gen)
    return x.to(dev), t.to(dev)


class Exact:
    def __init__(self, x, t, ignore=-100):
        x = x.double()
        m = x.amax(1, keepdim=True)
        m = torch.where(m == -math.inf, 0.0, m)
        e = torch.exp(x - m)
        self.z = e.sum(1, keepdim=True)
        self.p = torch.where(self.z > 0, e / self.z, 0.0)
        self.lp = x - m - torch.log(self.z)
        self.lp = torch.where(x == -math.inf, -math.inf, self.lp)
        flat = torch.where(self.p > 0, self.lp, 0.0)
        self.entropy = -(self.p * flat).sum(1)
        d = torch.where(self.p > 0, x - m, 0.0)
        self.d = d
        self.ed, self.ed2 = (self.p * d.abs()).sum(1), (self.p * d * d).sum(1)
        self.given = t != ignore
        self.at = t.clamp(0, x.shape[1] - 1)[:, None]
        self.logprob = torch.where(self.given, self.lp.gather(1, self.at)[:, 0], 0.0)

    def check(self, r):
        near = lambda a, b, tol: bool((((a.double() - b).abs() <= tol) | (a.double() == b)).all())
        off = E20 + E22 * self.ed
        assert r.logprobs.dtype == r.entropy.dtype == F32
        assert near(r.logprobs, self.logprob, off + 2.0 ** -23 * self.logprob.abs())
        assert near(r.entropy, self.entropy, 2 * off * (1 + self.ed) + E22 * self.ed2)

    def check_top(self, r, x, k):
        order = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :k]
        assert torch.equal(r.top_indices, order)
        ref = self.lp.gather(1, order)
        tol = (E20 + E22 * self.ed)[:, None] + 2.0 ** -23 * ref.abs()
        assert (((r.top_logprobs.double() - ref).abs() <= tol) | (r.top_logprobs == ref)).all()

    def check_grad(self, dx, gl, gh):
        gl = torch.where(self.given, gl.double(), 0.0)[:, None]
        gh = gh.double()[:, None]
        flat = torch.where(self.p > 0, self.lp, 0.0)
        ref = -gl * self.p - gh * self.p * (flat + self.entropy[:, None])
        ref = ref.scatter_add(1, self.at, gl)
        ent = self.entropy[:, None]
        rel = 4 * (E20 + E22 * (self.ed[:, None] + self.d.abs()))
        size = self.p * (gl.abs() + gh.abs() * (flat.abs() + ent + 1 + self.ed2[:, None]))
        bound = UNIT[dx.dtype] * ref.abs() + TINY[dx.dtype] + rel * size
        bound = bound.scatter_add(1, self.at, 2.0 ** -23 * gl.abs())
        assert ((dx.double() - ref).abs() <= bound).all()


SIZES = [(1, 1), (1, 2), (3, 7), (2, 8), (5, 33), (40, 257), (3, 4096), (900, 1000), (2, 32768), (1, 32769), (3, 50257),
         (1, 131072), (2, 200003), (600, 5001)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_forward_top_and_gradient(cuda_device, native_lib, rows, vocab, dtype):
    x, t = make(rows, vocab, dtype, cuda_device)
    ex = Exact(x, t)
    ex.check(logprobs.token_logprobs(x, t))
    for k in sorted({1, min(5, vocab), min(logprobs.MAX_TOP, vocab)}):
        r = logprobs.token_logprobs(x, t, top_k=k)
        ex.check(r)
        ex.check_top(r, x, k)
    leaf = x.clone().requires_grad_()
    r = logprobs.token_logprobs(leaf, t)
    gen = torch.Generator().manual_seed(vocab)
    gl, gh = (torch.randn(rows, generator=gen).to(cuda_device) for _ in range(2))
    dx, = torch.autograd.grad((r.logprobs, r.entropy), (leaf,), (gl, gh))
    ex.check_grad(dx, gl, gh)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [100, 5000, 70001])
def test_barred_tokens_and_empty_rows(cuda_device, native_lib, vocab):
    x, t = make(12, vocab, BF16, cuda_device, barred=0.5)
    x[4] = -math.inf                                     # nothing is left
    x[5] = -math.inf
    x[5, vocab - 3] = 1.5                                # one token is left
    t[5] = vocab - 3
    x[6, t[6]] = -math.inf                               # the given token is barred
    ex = Exact(x, t)
    k = min(vocab, 20)
    r = logprobs.token_logprobs(x, t, top_k=k)
    ex.check(r)
    ex.check_top(r, x, k)
    assert r.logprobs[4] == -math.inf and r.entropy[4] == 0
    assert r.logprobs[5] == 0 and r.entropy[5] == 0 and r.logprobs[6] == -math.inf
    leaf = x.clone().requires_grad_()
    q = logprobs.token_logprobs(leaf, t)
    t2 = t.clone()
    gl = torch.ones(12, device=cuda_device)
    dx, = torch.autograd.grad((q.logprobs, q.entropy), (leaf,), (gl, gl))
    assert dx.isfinite().all() and not dx[4].any()
    keep = [i for i in range(12) if i != 4]
    Exact(x[keep], t2[keep]).check_grad(dx[keep], gl[keep], gl[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("vocab", [1, 31, 300, 2050, 6144, 6145])
def test_many_short_rows(cuda_device, native_lib, vocab, dtype):
    """Rows of one warp each, and just past them: barred tokens, empty rows, an odd pitch, a given token left out."""
    rows = 1187
    x, t = make(rows, vocab + 3, dtype, cuda_device, barred=0.1)
    x, t = x[:, :vocab], t.clamp(max=vocab - 1)
    x[::50] = -math.inf
    t[7::40] = -100
    x[5] = 1.0                                           # all alike
    x[6] = torch.arange(vocab, device=cuda_device) % 2   # two values
    ex = Exact(x, t)
    ex.check(logprobs.token_logprobs(x, t))
    for k in sorted({min(k, vocab) for k in (1, 5, 16, 24, 25)}):
        r = logprobs.token_logprobs(x, t, top_k=k)
        ex.check(r)
        ex.check_top(r, x, k)
        bad = torch.empty_strided(x.shape, x.stride(), dtype=dtype, device=cuda_device).copy_(x)  # the same pitch
        bad[::3, vocab // 2] = math.nan
        q = logprobs.token_logprobs(bad, t, top_k=k)
        assert q.entropy[::3].isnan().all() and (q.top_indices[::3, 0] == vocab // 2).all()
        for a, b in ((q.logprobs, r.logprobs), (q.entropy, r.entropy), (q.top_indices, r.top_indices)):
            assert torch.equal(a[1::3], b[1::3]) and torch.equal(a[2::3], b[2::3])
    leaf = x.clone().requires_grad_()
    r = logprobs.token_logprobs(leaf, t)
    gen = torch.Generator().manual_seed(vocab)
    gl, gh = (torch.randn(rows, generator=gen).to(cuda_device) for _ in range(2))
    dx, = torch.autograd.grad((r.logprobs, r.entropy), (leaf,), (gl, gh))
    none = (x == -math.inf).all(1)
    assert not dx[none].any()
    Exact(x[~none], t[~none]).check_grad(dx[~none], gl[~none], gh[~none])


@pytest.mark.gpu
def test_lowest_value_masks(cuda_device, native_lib):
    """Masks written as the type's lowest value: probability 0, no overflow."""
    for dtype in (F16, BF16, F32):
        x, t = make(6, 3001, dtype, cuda_device)
        x[:, ::2] = torch.finfo(dtype).min
        x[3] = torch.finfo(dtype).min                    # a whole row: uniform
        t = t // 2 * 2 + 1
        t.clamp_(max=2999)
        ex = Exact(x, t)
        leaf = x.clone().requires_grad_()
        r = logprobs.token_logprobs(leaf, t, top_k=10)
        ex.check(r)
        ex.check_top(r, x, 10)
        g = torch.ones(6, device=cuda_device)
        dx, = torch.autograd.grad((r.logprobs, r.entropy), (leaf,), (g, g))
        ex.check_grad(dx, g, g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, F32])
def test_ties_go_to_the_lower_index(cuda_device, native_lib, dtype):
    gen = torch.Generator().manual_seed(3)
    for vocab in (50, 2049, 40000):
        x = torch.randint(-2, 3, (4, vocab), generator=gen).to(dtype).to(cuda_device)
        x[0] = 1.0
        x[1, ::3] = -0.0                                 # equals +0
        x[1, 1::3] = 0.0
        x[2] = torch.arange(vocab) // 50                 # ascending: every element beats those before
        t = torch.zeros(4, dtype=torch.long, device=cuda_device)
        r = logprobs.token_logprobs(x, t, top_k=40)
        Exact(x, t).check_top(r, x, 40)


@pytest.mark.gpu
def test_clustered_top(cuda_device, native_lib):
    """All the largest logits in one stretch, and all in one thread's share."""
    x, t = make(3, 30000, F32, cuda_device)
    x[0, 17000:17100] += 50
    x[1, 8 * torch.arange(0, 30000 // 8, 256)] += 50
    x[2, -5:] += 50
    r = logprobs.token_logprobs(x, t, top_k=64)
    Exact(x, t).check_top(r, x, 64)


@pytest.mark.gpu
def test_ignored_and_invalid_targets(cuda_device, native_lib):
    x, t = make(8, 600, F32, cuda_device)
    t[1], t[2], t[3], t[4] = -100, 600, -1, 2 ** 40
    leaf = x.clone().requires_grad_()
    r = logprobs.token_logprobs(leaf, t)
    assert r.logprobs[1] == 0 and r.logprobs[2:5].isnan().all()
    good = [0, 1, 5, 6, 7]
    gl = torch.randn(8, device=cuda_device)
    gh = torch.randn(8, device=cuda_device)
    dx, = torch.autograd.grad((r.logprobs, r.entropy), (leaf,), (gl, gh))
    ex = Exact(x[good], t[good])
    ex.check(logprobs.TokenLogprobs(r.logprobs[good], r.entropy[good], None, None))
    ex.check_grad(dx[good], gl[good], gh[good])
    r2 = logprobs.token_logprobs(x, torch.full((8,), 5, device=cuda_device), ignore_index=5)
    assert not r2.logprobs.any()


@pytest.mark.gpu
def test_one_gradient_only(cuda_device, native_lib):
    x, t = make(9, 777, BF16, cuda_device)
    ex, zero = Exact(x, t), torch.zeros(9, device=cuda_device)
    g = torch.randn(9, device=cuda_device)
    for which in range(2):
        leaf = x.clone().requires_grad_()
        out = logprobs.token_logprobs(leaf, t)[which]
        dx, = torch.autograd.grad(out, (leaf,), g)
        ex.check_grad(dx, g if which == 0 else zero, zero if which == 0 else g)


@pytest.mark.gpu
def test_nan_and_inf_stay_in_their_rows(cuda_device, native_lib):
    x, t = make(6, 5000, F16, cuda_device)
    x[1, 77], x[2, 88] = math.nan, math.inf
    t[1], t[2] = 0, 0
    r = logprobs.token_logprobs(x, t, top_k=3)
    assert r.logprobs[1].isnan() and r.entropy[1].isnan() and r.logprobs[2].isnan()
    assert r.top_indices[1, 0] == 77 and r.top_indices[2, 0] == 88
    good = [0, 3, 4, 5]
    Exact(x[good], t[good]).check(logprobs.TokenLogprobs(r.logprobs[good], r.entropy[good], None, None))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, F32])
def test_layouts(cuda_device, native_lib, dtype):
    x0, t = make(10, 700, dtype, cuda_device)
    for view in (x0[:, 3:603], x0[:, 8:608], x0[::2, :600], x0.t().contiguous().t()[:, :601],
                 x0[:1].expand(10, 700)[:, :600]):
        n, v = view.shape
        tt = t[:n].clamp(max=v - 1)
        ex = Exact(view, tt)
        r = logprobs.token_logprobs(view, tt, top_k=7)
        ex.check(r)
        ex.check_top(r, view, 7)
        leaf = view.detach().requires_grad_()
        g = torch.randn(n, device=cuda_device)
        q = logprobs.token_logprobs(leaf, tt)
        dx, = torch.autograd.grad((q.logprobs, q.entropy), (leaf,), (g, g))
        ex.check_grad(dx, g, g)
    x3, t3 = x0[:, :600].reshape(2, 5, 600), (t % 600).view(2, 5).int()
    r = logprobs.token_logprobs(x3, t3, top_k=2)
    assert r.logprobs.shape == (2, 5) and r.top_indices.shape == (2, 5, 2)
    Exact(x3.view(10, 600), t3.view(10).long()).check(
        logprobs.TokenLogprobs(r.logprobs.view(10), r.entropy.view(10), None, None))


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda_device, native_lib):
    """Rows that start beyond 2^32 elements."""
    rows, vocab, ld = 3, 300, 2 ** 31 + 8
    base = torch.empty((rows - 1) * ld + vocab, dtype=F16, device=cuda_device)
    x0, t = make(rows, vocab, F16, cuda_device)
    x = base.as_strided((rows, vocab), (ld, 1))
    x.copy_(x0)
    r = logprobs.token_logprobs(x, t, top_k=4)
    ex = Exact(x0, t)
    ex.check(r)
    ex.check_top(r, x0, 4)


@pytest.mark.gpu
def test_gradient_against_differences(cuda_device, native_lib):
    """<dx, v> against the central difference along v in 64 bits (step 1e-4: error about 1e-8)."""
    x, t = make(5, 60, F32, cuda_device, std=1.5)
    gen = torch.Generator().manual_seed(1)
    gl, gh = (torch.randn(5, generator=gen).to(cuda_device) for _ in range(2))
    v = torch.randn(x.shape, generator=gen).to(cuda_device).double()
    leaf = x.clone().requires_grad_()
    r = logprobs.token_logprobs(leaf, t)
    dx, = torch.autograd.grad((r.logprobs, r.entropy), (leaf,), (gl, gh))
    def f(s):
        ex = Exact(x.double() + s * v, t)
        return (gl * ex.logprob + gh * ex.entropy).sum()
    diff = (f(1e-4) - f(-1e-4)) / 2e-4
    assert abs((dx.double() * v).sum() - diff) <= 1e-5 * (dx.double() * v).abs().sum() + 1e-6


@pytest.mark.gpu
def test_empty_stream_graph_and_operator(cuda_device, native_lib):
    none = torch.zeros(0, dtype=torch.long, device=cuda_device)
    r = logprobs.token_logprobs(torch.zeros((0, 9), device=cuda_device), none, top_k=2)
    assert r.logprobs.shape == (0,) and r.top_indices.shape == (0, 2)
    x, t = make(3, 90000, F32, cuda_device)
    ex = Exact(x, t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = x * 1.0
        q = logprobs.token_logprobs(y, t, top_k=5)
    s.synchronize()
    ex.check(q)
    ex.check_top(q, x, 5)
    graph = torch.cuda.CUDAGraph()
    buf = torch.zeros_like(x)
    with torch.cuda.graph(graph):
        out = logprobs.token_logprobs(buf, t, top_k=5)
    buf.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    ex.check(out)
    ex.check_top(out, x, 5)
    leaf = x[:, :50].clone().requires_grad_()
    lp, ent, *_ = torch.ops.tensorcore_gemm.token_logprobs(leaf, t % 50, 3, -100)
    g = torch.ones(3, device=cuda_device)
    dx, = torch.autograd.grad((lp, ent), (leaf,), (g, g))
    Exact(leaf.detach(), t % 50).check_grad(dx, g, g)
    torch.library.opcheck(torch.ops.tensorcore_gemm.token_logprobs, (leaf, t % 50, 3, -100),
                          test_utils=("test_schema", "test_faketensor"))


@pytest.mark.gpu
def test_refusals(cuda_device, native_lib):
    x = torch.zeros((4, 16), device=cuda_device)
    t = torch.zeros(4, dtype=torch.long, device=cuda_device)
    for args, kw, match in [((x.double(), t), {}, "logits must be"), ((x, t.float()), {}, "targets must be"),
                            ((x, t[:3]), {}, "shape"), ((x, t), {"top_k": 17}, "top_k"),
                            ((x, t), {"top_k": -1}, "top_k"), ((x, t.cpu()), {}, "CUDA"), ((x[:, :0], t), {}, "at least one")]:
        with pytest.raises(RuntimeError, match=match):
            logprobs.token_logprobs(*args, **kw)
    wide = torch.zeros((1, 100), device=cuda_device)
    with pytest.raises(RuntimeError, match="top_k"):
        logprobs.token_logprobs(wide, t[:1], top_k=logprobs.MAX_TOP + 1)


def test_cpu_tensors_raise():
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        logprobs.token_logprobs(torch.zeros((4, 16)), torch.zeros(4, dtype=torch.long))


def test_fake_shapes_without_gpu():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode(allow_non_fake_inputs=False):
        x = torch.empty((3, 5, 80), dtype=BF16, device="cuda")
        t = torch.empty((3, 5), dtype=torch.long, device="cuda")
        r = logprobs.token_logprobs(x, t, top_k=4)
        assert r.logprobs.shape == (3, 5) and r.top_logprobs.shape == (3, 5, 4) and r.top_indices.dtype == torch.int64
        assert logprobs.token_logprobs(x, t).top_indices is None


def test_c_argument_checks_without_gpu(native_lib):
    size, fwd, bwd = (native_lib.b200_token_logprobs_workspace_size, native_lib.b200_token_logprobs_fwd,
                      native_lib.b200_token_logprobs_bwd)
    p = 4096
    assert size(1000, 1000, 5) == 0 and size(1, 131072, 5) > 0 and size(1, 8, 65) == -1 and size(1, 1 << 31, 0) == -3
    args = [p] * 7 + [4, 100, 100, 2, -100, 0, None, 0, None]
    def with_(i, v):
        return [v if j == i else a for j, a in enumerate(args)]
    for i, v in [(0, None), (1, None), (2, None), (3, None), (5, None), (6, None), (7, -1), (8, 0), (9, 99), (10, 65),
                 (12, 3)]:
        assert fwd(*with_(i, v)) == 1, i
    assert fwd(*with_(8, 1 << 31)) == 3
    assert fwd(*with_(7, 0)) == 0
    big = [p] * 7 + [1, 131072, 131072, 5, -100, 0, p + 8, 1 << 20, None]
    assert fwd(*big) == 8                                   # misaligned workspace
    assert bwd(p, p, p, p, p, p, None, 4, 100, 100, 100, -100, 0, None) == 1
    assert bwd(p, p, p, p, p, p, p, 4, 100, 99, 100, -100, 0, None) == 1


# Stretches of a row that are masked, as (first, last) of the vocabulary's length.
STRETCHES = [(0.0, 0.05), (0.95, 1.0), (0.4, 0.6), (0.0, 0.5), (0.5, 1.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,vocab", [(7, 300), (1187, 300), (7, 5000), (1187, 5000), (7, 50257), (7, 200003)])
def test_masked_stretches(cuda_device, native_lib, rows, vocab, dtype):
    """Contiguous masks of finite lowest values: padded vocabularies, constrained decoding."""
    masks = [torch.finfo(dtype).min] if dtype == F16 else [torch.finfo(dtype).min, -1e38, -1e31, -2e30]
    for mask in masks:
        x, t = make(rows, vocab, dtype, cuda_device)
        for i in range(rows):
            if i % 7 < 5:
                lo, hi = STRETCHES[i % 7]
                x[i, round(lo * vocab):round(hi * vocab)] = mask
            elif i % 7 == 5:                             # all but three logits
                keep = x[i, [1, vocab // 2, vocab - 2]].clone()
                x[i] = mask
                x[i, [1, vocab // 2, vocab - 2]] = keep
                t[i] = vocab // 2
            else:                                        # a mixture of masks, one stretch each
                x[i, :vocab // 3] = mask
                x[i, vocab // 3:2 * vocab // 3] = -math.inf
                t[i] = vocab - 1
        ex = Exact(x, t)
        ex.check(logprobs.token_logprobs(x, t))
        for k in (1, 20, 40):
            r = logprobs.token_logprobs(x, t, top_k=k)
            ex.check(r)
            ex.check_top(r, x, k)
        leaf = x.clone().requires_grad_()
        r = logprobs.token_logprobs(leaf, t)
        gl, gh = (torch.randn(rows, device=cuda_device) for _ in range(2))
        dx, = torch.autograd.grad((r.logprobs, r.entropy), (leaf,), (gl, gh))
        ex.check_grad(dx, gl, gh)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,vocab", [(4, 300), (1187, 300), (4, 50257), (4, 200003)])
def test_forced_token(cuda_device, native_lib, rows, vocab, dtype):
    """One logit at the type's highest value: it has all the probability, wherever it stands."""
    x, t = make(rows, vocab, dtype, cuda_device)
    at = torch.arange(rows, device=cuda_device) * 97 % vocab
    at[:4] = torch.tensor([0, vocab - 1, vocab // 2, 9], device=cuda_device)
    x[torch.arange(rows, device=cuda_device), at] = torch.finfo(dtype).max
    t[::2] = at[::2]
    ex = Exact(x, t)
    r = logprobs.token_logprobs(x, t, top_k=3)
    ex.check(r)
    ex.check_top(r, x, 3)
    ex.check(logprobs.token_logprobs(x, t))
    leaf = x.clone().requires_grad_()
    q = logprobs.token_logprobs(leaf, t)
    gl, gh = (torch.randn(rows, device=cuda_device) for _ in range(2))
    dx, = torch.autograd.grad((q.logprobs, q.entropy), (leaf,), (gl, gh))
    ex.check_grad(dx, gl, gh)


@pytest.mark.gpu
def test_backward_operator_refusals(cuda_device, native_lib):
    """The backward operator refuses what its kernels would read out of range."""
    op = torch.ops.tensorcore_gemm.token_logprobs_backward
    x, t = make(6, 90, BF16, cuda_device)
    _, ent, stats, *_ = torch.ops.tensorcore_gemm.token_logprobs(x, t, 0, -100)
    g = torch.randn(6, device=cuda_device)
    Exact(x, t).check_grad(op(x, t, stats, ent, g, g, -100), g, g)
    Exact(x, t).check_grad(op(x, t, stats.t().contiguous().t(), ent, g, None, -100), g, 0 * g)
    for args, match in [((x, t, stats[:3], ent, g, g), "stats must have shape"), ((x, t, stats.double(), ent, g, g), "stats must be"),
                        ((x, t, stats, ent[:3], g, g), "entropy must"), ((x, t, stats, ent, g[:3], g), "g_logprob must"),
                        ((x, t, stats, ent, g, g.half()), "g_entropy must"), ((x, t, stats, ent, None, g[:1]), "g_entropy must"),
                        ((x, t[:3], stats, ent, g, g), "shape"), ((x, t, stats.cpu(), ent, g, g), "CUDA"),
                        ((x.double(), t, stats, ent, g, g), "logits must")]:
        with pytest.raises(RuntimeError, match=match):
            op(*args, -100)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(6, 600), (6, 40000), (1300, 600)])
def test_invalid_targets_have_no_finite_gradient(cuda_device, native_lib, rows, vocab):
    """The gradient of a NaN log probability is NaN, not that of -lse; rows that do not use it are as they were."""
    x, t = make(rows, vocab, F32, cuda_device)
    t[1], t[2], t[3], t[4] = vocab, -1, 2 ** 40, -1
    gl, gh = (torch.randn(rows, device=cuda_device) for _ in range(2))
    gl[4] = 0.0
    leaf = x.clone().requires_grad_()
    r = logprobs.token_logprobs(leaf, t)
    dx, = torch.autograd.grad((r.logprobs, r.entropy), (leaf,), (gl, gh), retain_graph=True)
    assert r.logprobs[1:5].isnan().all() and dx[1:4].isnan().all()
    t2 = t.clone()
    t2[4] = -100
    good = [i for i in range(rows) if i not in (1, 2, 3)]
    Exact(x[good], t2[good]).check_grad(dx[good], gl[good], gh[good])
    dx, = torch.autograd.grad(r.entropy, (leaf,), gh)
    t2[1:5] = -100
    Exact(x, t2).check_grad(dx, 0 * gl, gh)
