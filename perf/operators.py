"""The language-model operators around the GEMM, as cases that can be run and timed.

Three operators of a transformer's feed-forward sublayer and of its head, forward and backward:

  norm    layer norm over the last dimension, with the gradients of its input, weight and bias
  ffn     the gated feed-forward block  y = (act(x Wg^T) * (x Wu^T)) Wo^T,  w_in = [Wg; Wu]
  lprob   log probabilities of given tokens, the entropy of their distributions and the
          top alternatives, with the gradient of the logits

`run` computes them in their plain form (elementary torch operations in 32 bits, rounded once),
or, where `own` is true, through this package's entry points.  `exact` restates them in 64 bits.
"""
import math
import sys
from pathlib import Path

import torch

own = False

IGNORE = -100
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # The norm before a block while tokens are generated: a handful of rows, latency counts.
        {"name": "norm decode", "op": "norm", "rows": 8, "cols": 4096, "dtype": "fp16", "wdtype": "fp16", "train": False},
        # The same norm over a batch of prompts of different lengths, packed.
        {"name": "norm prompts", "op": "norm", "rows": 20011, "cols": 5120, "dtype": "bf16", "wdtype": "bf16", "train": False},
        # A training step's norm: activations in 16 bits, weight and bias kept in 32.
        {"name": "norm train", "op": "norm", "rows": 16384, "cols": 4096, "dtype": "bf16", "wdtype": "fp32", "train": True},
        # A small model with an odd width, trained in 32 bits (no row starts on 16 bytes).
        {"name": "norm train odd", "op": "norm", "rows": 2999, "cols": 771, "dtype": "fp32", "wdtype": "fp32", "train": True},
        # One token of one request through the block: bound by reading the weights.
        {"name": "ffn decode 1", "op": "ffn", "rows": 1, "dim": 4096, "hidden": 12288, "act": "silu", "dtype": "fp16", "train": False},
        # A step of a batch of requests on a smaller model.
        {"name": "ffn decode 24", "op": "ffn", "rows": 24, "dim": 2048, "hidden": 5504, "act": "gelu_tanh", "dtype": "bf16", "train": False},
        # Packed prompts.
        {"name": "ffn prompts", "op": "ffn", "rows": 4001, "dim": 4096, "hidden": 12288, "act": "silu", "dtype": "fp16", "train": False},
        # A training step of the block.
        {"name": "ffn train", "op": "ffn", "rows": 8192, "dim": 4096, "hidden": 11008, "act": "silu", "dtype": "bf16", "train": True},
        # A small model with sizes that no tile divides.
        {"name": "ffn train odd", "op": "ffn", "rows": 1111, "dim": 1000, "hidden": 2731, "act": "gelu", "dtype": "fp16", "train": True},
        # Log probabilities beside sampled tokens, with the alternatives a server returns.
        {"name": "lprob decode", "op": "lprob", "rows": 7, "vocab": 131072, "top": 20, "dtype": "fp32", "train": False},
        # Scoring given texts.
        {"name": "lprob score", "op": "lprob", "rows": 4096, "vocab": 50257, "top": 5, "dtype": "bf16", "train": False},
        # The loss and an entropy bonus of a training step, with the gradient of the logits.
        {"name": "lprob train", "op": "lprob", "rows": 8192, "vocab": 65536, "top": 0, "dtype": "bf16", "train": True},
    ]


def _log_int(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm; one in two is rounded to a multiple of 8."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v > 16 and rng.random() < 0.5:
        v -= v % 8
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["norm", "ffn", "lprob"])
    train = rng.random() < 0.5
    if op == "norm":
        cols = _log_int(rng, 64, 16384)
        rows = _log_int(rng, 1, max(1, min(65536, 16384 * 4096 // cols)))
        dtype = rng.choice(["fp16", "bf16", "fp32"])
        if dtype == "fp32":
            rows = max(1, rows // 2)
        return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "wdtype": rng.choice([dtype, "fp32"]), "train": train}
    if op == "ffn":
        dim = _log_int(rng, 128, 4096)
        hidden = min(11008, max(128, int(dim * rng.uniform(2.0, 4.0))))
        rows = _log_int(rng, 1, 8192 if rng.random() < 0.7 else 64)
        return {"op": op, "rows": rows, "dim": dim, "hidden": hidden, "act": rng.choice(["silu", "gelu", "gelu_tanh"]),
                "dtype": rng.choice(["fp16", "bf16"]), "train": train}
    vocab = _log_int(rng, 256, 131072)
    dtype = rng.choice(["fp16", "bf16", "fp32"])
    most = 8192 * 65536 // vocab // (2 if dtype == "fp32" else 1)
    rows = _log_int(rng, 1, min(8192, most))
    top = 0 if train else rng.choice([0, 1, 5, 20])
    if top:
        rows = min(rows, max(1, 4096 * 50257 // vocab))
    return {"op": op, "rows": rows, "vocab": vocab, "top": top, "dtype": dtype, "train": train}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _normal(gen, shape, std, dtype, mean=0.0):
    t = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return t.mul_(std).add_(mean).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        # A residual stream: a mean that differs from row to row, and some channels far larger than the rest.
        x = torch.randn((rows, cols), generator=gen, device="cuda")
        loud = torch.rand((cols,), generator=gen, device="cuda") < 0.01
        x *= torch.where(loud, 8.0, 1.0)
        x += 0.5 * torch.randn((rows, 1), generator=gen, device="cuda")
        s["x"] = x.to(dt)
        s["weight"] = _normal(gen, (cols,), 0.1, DTYPES[case["wdtype"]], 1.0)
        s["bias"] = _normal(gen, (cols,), 0.1, DTYPES[case["wdtype"]])
        if case["train"]:
            s["grad"] = _normal(gen, (rows, cols), 1.0, dt)
        leaves = ("x", "weight", "bias")
    elif case["op"] == "ffn":
        rows, dim, hidden = case["rows"], case["dim"], case["hidden"]
        s["x"] = _normal(gen, (rows, dim), 1.0, dt)
        s["w_in"] = _normal(gen, (2 * hidden, dim), dim ** -0.5, dt)
        s["w_out"] = _normal(gen, (dim, hidden), hidden ** -0.5, dt)
        if case["train"]:
            s["grad"] = _normal(gen, (rows, dim), 1.0, dt)
        leaves = ("x", "w_in", "w_out")
    else:
        rows, vocab = case["rows"], case["vocab"]
        s["logits"] = _normal(gen, (rows, vocab), 3.0, dt)
        s["targets"] = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        if case["train"]:
            # Padding in the batch has no target; policy-gradient weights on the rest.
            pad = torch.rand((rows,), generator=gen, device="cuda") < 0.05
            s["targets"] = torch.where(pad, IGNORE, s["targets"])
            s["grad_logprob"] = _normal(gen, (rows,), 1.0, torch.float32)
            s["grad_entropy"] = _normal(gen, (rows,), 0.1, torch.float32)
        else:
            # A server bars some tokens (their logits are -inf), though not the given one.
            barred = torch.rand((vocab,), generator=gen, device="cuda") < 0.02
            kept = s["logits"].gather(1, s["targets"][:, None])
            s["logits"].masked_fill_(barred[None, :], -math.inf)
            s["logits"].scatter_(1, s["targets"][:, None], kept)
        leaves = ("logits",)
    if case["train"]:
        for name in leaves:
            s[name].requires_grad_()
    return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _act(kind, g):
    """act(g) and its derivative."""
    if kind == "silu":
        sig = 1 / (1 + torch.exp(-g))
        return g * sig, sig * (1 + g * (1 - sig))
    if kind == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    c, a = math.sqrt(2 / math.pi), 0.044715
    t = torch.tanh(c * (g + a * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * a * g * g)


def _norm(s, wide):
    x, w, b = s["x"].detach().to(wide), s["weight"].detach().to(wide), s["bias"].detach().to(wide)
    d = x - x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5)
    xhat = d * rstd
    out = {"y": xhat * w + b}
    if s["train"]:
        dy = s["grad"].to(wide)
        dxhat = dy * w
        out["dx"] = rstd * (dxhat - dxhat.mean(1, keepdim=True) - xhat * (dxhat * xhat).mean(1, keepdim=True))
        out["dweight"] = (dy * xhat).sum(0)
        out["dbias"] = dy.sum(0)
    return out


def _ffn(s, wide):
    x, w_in, w_out = s["x"].detach().to(wide), s["w_in"].detach().to(wide), s["w_out"].detach().to(wide)
    h = w_out.shape[1]
    gu = x @ w_in.t()
    g, u = gu[:, :h], gu[:, h:]
    act, slope = _act(s["act"], g)
    out = {"y": (act * u) @ w_out.t()}
    if s["train"]:
        dy = s["grad"].to(wide)
        da = dy @ w_out
        dgu = torch.cat([da * u * slope, da * act], 1)
        out["dx"] = dgu @ w_in
        out["dw_in"] = dgu.t() @ x
        out["dw_out"] = dy.t() @ (act * u)
    return out


def _sort_keys(logits32):
    """Whole numbers that order as (value, then lower index first): no two of a row are alike."""
    bits = logits32.view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
    n = logits32.shape[1]
    return (order << 32) + torch.arange(n - 1, -1, -1, device=logits32.device)


def _lprob(s, wide):
    x, t = s["logits"].detach().to(wide), s["targets"]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    lse = m + torch.log(z)
    p, lp = e / z, x - lse
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
    given = t >= 0
    at = t.clamp(min=0)[:, None]
    out = {"logprob": torch.where(given, lp.gather(1, at)[:, 0], torch.zeros_like(ent)), "entropy": ent}
    if s["top"]:
        keys = _sort_keys(s["logits"].detach().float())
        out["top_indices"] = torch.topk(keys, s["top"], 1).indices
        out["top_logprobs"] = lp.gather(1, out["top_indices"])
    if s["train"]:
        gl = torch.where(given, s["grad_logprob"].to(wide), 0)[:, None]
        ge = s["grad_entropy"].to(wide)[:, None]
        d = -gl * p - ge * torch.where(p > 0, p * (lp + ent[:, None]), torch.zeros_like(p))
        out["dlogits"] = d.scatter_add_(1, at, gl)
    return out


def _rounded(s, out):
    """Each output rounded once, to the type that the operator gives it."""
    kinds = {"y": "x", "dx": "x", "dweight": "weight", "dbias": "bias", "dw_in": "w_in", "dw_out": "w_out", "dlogits": "logits"}
    return {k: v.to(s[kinds[k]].dtype) if k in kinds else v if k == "top_indices" else v.to(torch.float32) for k, v in out.items()}


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _package():
    home = str(Path(__file__).resolve().parent.parent / "ampere-gemm_b200")
    if home not in sys.path:
        sys.path.insert(0, home)
    from tensorcore_gemm import ffn, logprobs, norm

    return norm, ffn, logprobs


def _run_own(s):
    norm, ffn, logprobs = _package()
    if s["op"] == "norm":
        out = {"y": norm.layer_norm(s["x"], s["weight"], s["bias"], eps=1e-5)}
        if s["train"]:
            out["dx"], out["dweight"], out["dbias"] = torch.autograd.grad(out["y"], (s["x"], s["weight"], s["bias"]), s["grad"])
    elif s["op"] == "ffn":
        out = {"y": ffn.gated_ffn(s["x"], s["w_in"], s["w_out"], activation=s["act"])}
        if s["train"]:
            out["dx"], out["dw_in"], out["dw_out"] = torch.autograd.grad(out["y"], (s["x"], s["w_in"], s["w_out"]), s["grad"])
    else:
        r = logprobs.token_logprobs(s["logits"], s["targets"], top_k=s["top"], ignore_index=IGNORE)
        out = {"logprob": r.logprobs, "entropy": r.entropy}
        if s["top"]:
            out["top_indices"], out["top_logprobs"] = r.top_indices, r.top_logprobs
        if s["train"]:
            out["dlogits"], = torch.autograd.grad((r.logprobs, r.entropy), (s["logits"],), (s["grad_logprob"], s["grad_entropy"]))
    return {k: v.detach() for k, v in out.items()}


def run(s):
    if own:
        return _run_own(s)
    plain = {"norm": _norm, "ffn": _ffn, "lprob": _lprob}[s["op"]]
    return _rounded(s, plain(s, torch.float32))


# ---------------------------------------------------------------------------
# What a pass cannot do without, and its exact outputs
# ---------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        # x in, y out; backward dy and x in, dx out.
        return {"bytes": n * size * (5 if case["train"] else 2), "flops": n * (20 if case["train"] else 8)}
    if case["op"] == "ffn":
        rows, dim, hidden = case["rows"], case["dim"], case["hidden"]
        weights = 3 * dim * hidden * size
        rows_b = rows * dim * size
        if case["train"]:
            # Forward: x, weights in, y out.  Backward: dy, x, weights in, dx and the weights' gradients out.
            return {"bytes": 3 * weights + 5 * rows_b, "flops": 18 * rows * dim * hidden}
        return {"bytes": weights + 2 * rows_b, "flops": 6 * rows * dim * hidden}
    n = case["rows"] * case["vocab"]
    # Logits in once; backward logits in, their gradient out.
    return {"bytes": n * size * (3 if case["train"] else 1), "flops": n * (14 if case["train"] else 6)}


def _exact_norm(s):
    x = s["x"].detach().double()
    w, b = s["weight"].detach().double(), s["bias"].detach().double()
    n = x.shape[1]
    mean = x.sum(1) / n
    centred = x - mean[:, None]
    dev = torch.sqrt(centred.pow(2).sum(1) / n + 1e-5)
    out = {"y": centred / dev[:, None] * w + b}
    if s["train"]:
        dy = s["grad"].double()
        h = centred / dev[:, None]
        q = dy * w
        # The Jacobian (I - 1 1^T / n - h h^T / n) / dev applied to q.
        out["dx"] = (q - q.sum(1, keepdim=True) / n - h * ((q * h).sum(1, keepdim=True) / n)) / dev[:, None]
        out["dweight"] = torch.einsum("ij,ij->j", dy, h)
        out["dbias"] = dy.sum(0)
    return out


def _exact_act(kind, g):
    if kind == "silu":
        sg = torch.sigmoid(g)
        return g * sg, sg + g * sg * torch.sigmoid(-g)
    if kind == "gelu":
        cdf = torch.special.ndtr(g)
        return g * cdf, cdf + g * torch.exp(-g.square() / 2) / math.sqrt(2 * math.pi)
    z = math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    sg = torch.sigmoid(2 * z)                      # (1 + tanh z) / 2
    return g * sg, sg + g * 2 * sg * torch.sigmoid(-2 * z) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g ** 2)


def _exact_ffn(s):
    x, w_out = s["x"].detach().double(), s["w_out"].detach().double()
    wg, wu = s["w_in"].detach().double().chunk(2, 0)
    g, u = x @ wg.t(), x @ wu.t()
    act, slope = _exact_act(s["act"], g)
    a = act * u
    out = {"y": a @ w_out.t()}
    if s["train"]:
        dy = s["grad"].double()
        da = dy @ w_out
        du, dg = da * act, da * u * slope
        out["dx"] = dg @ wg + du @ wu
        out["dw_in"] = torch.cat([dg.t() @ x, du.t() @ x], 0)
        out["dw_out"] = dy.t() @ a
    return out


def _exact_lprob(s):
    parts = []
    for i in range(0, s["rows"], 1024):
        x = s["logits"][i:i + 1024].detach().double()
        t = s["targets"][i:i + 1024]
        lp = torch.log_softmax(x, 1)
        p = lp.exp()
        ent = torch.special.entr(p).sum(1)
        given = t >= 0
        at = t.clamp(min=0)[:, None]
        out = {"logprob": torch.where(given, lp.gather(1, at)[:, 0], 0.0), "entropy": ent}
        if s["top"]:
            v, order = torch.sort(x, dim=1, descending=True, stable=True)
            out["top_indices"] = order[:, :s["top"]].clone()
            out["top_logprobs"] = lp.gather(1, out["top_indices"])
        if s["train"]:
            gl = torch.where(given, s["grad_logprob"][i:i + 1024].double(), 0.0)[:, None]
            ge = s["grad_entropy"][i:i + 1024].double()[:, None]
            one = torch.zeros_like(p).scatter_(1, at, 1.0)
            # d entropy / d x_j = -p_j (log p_j + entropy) = entr(p_j) - p_j entropy
            out["dlogits"] = gl * (one - p) + ge * (torch.special.entr(p) - p * ent[:, None])
        parts.append(out)
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "ffn": _exact_ffn, "lprob": _exact_lprob}[case["op"]](s)
