"""Log probabilities of given tokens, with entropies and top alternatives.

For a row x of logits and its target t, with lse = ln sum exp(x):

    logprob = x_t - lse
    entropy = -sum p ln p,  p = exp(x - lse)
    d logprob / d x_j = [j == t] - p_j
    d entropy / d x_j = -p_j (x_j - lse + entropy)

`token_logprobs` is the entry point; `torch.ops.tensorcore_gemm.token_logprobs`
is the same operator for tracers (it also returns the rows' statistics).  The
logits are read once, all sums are in fp32.  CUDA tensors only; nothing falls
back to another implementation.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _native
from ._rows import (DTYPE_CODES, as_rows, check_cuda, check_operand, launch, once_differentiable, plain_eager, ptr,
                    refuse_tangents, wants_grad, workspace)

#: Most alternatives a call can ask for.
MAX_TOP = _native.B200_LOGPROBS_MAX_TOP


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor                 # float32, the targets' shape
    entropy: torch.Tensor                  # float32, the targets' shape
    top_logprobs: Optional[torch.Tensor]   # float32, (..., top_k), largest first
    top_indices: Optional[torch.Tensor]    # int64, (..., top_k)


def _check(logits, targets, top_k: int) -> None:
    check_cuda("logits", logits)
    check_cuda("targets", targets, (torch.int64, torch.int32))
    if logits.dim() < 1 or logits.shape[:-1] != targets.shape:
        raise RuntimeError("targets must have logits' shape without its last dimension")
    if targets.device != logits.device:
        raise RuntimeError("logits and targets must be on the same CUDA device")
    if logits.shape[-1] == 0:
        raise RuntimeError("logits need at least one token")
    if not 0 <= top_k <= min(MAX_TOP, logits.shape[-1]):
        raise RuntimeError(f"top_k must be between 0 and {min(MAX_TOP, logits.shape[-1])}")


def _targets(t):
    return t.contiguous() if t.dtype == torch.int64 else t.to(torch.int64).contiguous()


def _forward(logits, targets, top_k: int, ignore_index: int, stats: bool = True):
    """logprobs, entropy, stats (..., 2) for the backward pass, top_logprobs and top_indices (..., top_k).

    None in the place of stats when they are not wanted, and of the last two for top_k = 0."""
    shape, dev = targets.shape, logits.device
    logprob = torch.empty(shape, dtype=torch.float32, device=dev)
    entropy = torch.empty_like(logprob)
    stats = torch.empty((*shape, 2), dtype=torch.float32, device=dev) if stats else None
    top_logprob = torch.empty((*shape, top_k), dtype=torch.float32, device=dev) if top_k else None
    top_index = torch.empty((*shape, top_k), dtype=torch.int64, device=dev) if top_k else None
    rows, vocab = targets.numel(), logits.shape[-1]
    if rows:
        x, ld = as_rows(logits)
        t = _targets(targets)
        ws_bytes = _native.load().b200_token_logprobs_workspace_size(rows, vocab, top_k)
        ws = workspace(ws_bytes, dev, "b200_token_logprobs_workspace_size")
        launch("b200_token_logprobs_fwd", logits.get_device(), x.data_ptr(), t.data_ptr(), logprob.data_ptr(),
               entropy.data_ptr(), ptr(stats), ptr(top_logprob), ptr(top_index), rows, vocab, ld, top_k,
               ignore_index, DTYPE_CODES[logits.dtype], ptr(ws), ws_bytes)
    return logprob, entropy, stats, top_logprob, top_index


def _backward(logits, targets, stats, entropy, g_logprob, g_entropy, ignore_index: int):
    d = torch.empty_like(logits, memory_format=torch.contiguous_format)
    rows, vocab = targets.numel(), logits.shape[-1]
    if rows:
        x, ld = as_rows(logits)
        t = _targets(targets)
        gl = None if g_logprob is None else g_logprob.contiguous()
        gh = None if g_entropy is None else g_entropy.contiguous()
        launch("b200_token_logprobs_bwd", logits.get_device(), x.data_ptr(), t.data_ptr(), stats.data_ptr(),
               entropy.data_ptr(), ptr(gl), ptr(gh), d.data_ptr(), rows, vocab, ld, vocab, ignore_index,
               DTYPE_CODES[logits.dtype])
    return d


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top_k, ignore_index):
        ctx.set_materialize_grads(False)
        logprob, entropy, stats, top_logprob, top_index = _forward(logits, targets, top_k, ignore_index)
        ctx.save_for_backward(logits, targets, stats, entropy)
        ctx.ignore_index = ignore_index
        if top_k:
            ctx.mark_non_differentiable(top_logprob, top_index)
        return logprob, entropy, top_logprob, top_index

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logprob, g_entropy, _g_top, _g_index):
        logits, targets, stats, entropy = ctx.saved_tensors
        eager = plain_eager(g_logprob, g_entropy)
        backward = _backward if eager else torch.ops.tensorcore_gemm.token_logprobs_backward
        return backward(logits, targets, stats, entropy, g_logprob, g_entropy, ctx.ignore_index), None, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top_k: int = 0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities of `targets` (...) under `logits` (..., V).

    logits are float16, bfloat16 or float32 (rows may be strided); targets are
    int64 or int32.  Also gives each row's entropy and, for top_k > 0 (at most
    MAX_TOP), the top_k largest log probabilities with their indices, equal
    logits by lower index.  A target equal to ignore_index has log probability
    0 and no gradient through it; another one outside [0, V) gives NaN, and a
    NaN gradient to its row unless the log probability's is 0.  A row of -inf
    throughout has log probability -inf, entropy 0 and gradient 0.
    Differentiable in the logits through logprobs and entropy (once); the
    alternatives are not differentiable.
    """
    if not plain_eager(logits, targets):
        lp, ent, _, tv, ti = torch.ops.tensorcore_gemm.token_logprobs(logits, targets, top_k, ignore_index)
    else:
        _check(logits, targets, top_k)
        if wants_grad(logits):
            lp, ent, tv, ti = _TokenLogprobs.apply(logits, targets, top_k, ignore_index)
        else:
            lp, ent, _, tv, ti = _forward(logits, targets, top_k, ignore_index, False)
    return TokenLogprobs(lp, ent, tv if top_k else None, ti if top_k else None)


# ---------------------------------------------------------------------------
# The dispatcher operators
# ---------------------------------------------------------------------------
@torch.library.custom_op("tensorcore_gemm::token_logprobs", mutates_args=())
def _token_logprobs_op(
        logits: torch.Tensor, targets: torch.Tensor, top_k: int,
        ignore_index: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """logprobs, entropy, stats, top_logprobs, top_indices (the last three are not differentiable)."""
    _check(logits, targets, top_k)
    refuse_tangents(logits)
    lp, ent, stats, tv, ti = _forward(logits, targets, top_k, ignore_index)
    if not top_k:
        tv, ti = (torch.empty((*targets.shape, 0), dtype=d, device=logits.device) for d in (torch.float32, torch.int64))
    return lp, ent, stats, tv, ti


@_token_logprobs_op.register_fake
def _(logits, targets, top_k, ignore_index):
    _check(logits, targets, top_k)
    shape, dev = targets.shape, logits.device
    return (torch.empty(shape, dtype=torch.float32, device=dev), torch.empty(shape, dtype=torch.float32, device=dev),
            torch.empty((*shape, 2), dtype=torch.float32, device=dev),
            torch.empty((*shape, top_k), dtype=torch.float32, device=dev),
            torch.empty((*shape, top_k), dtype=torch.int64, device=dev))


@torch.library.custom_op("tensorcore_gemm::token_logprobs_backward", mutates_args=())
def _token_logprobs_backward_op(logits: torch.Tensor, targets: torch.Tensor, stats: torch.Tensor,
                                entropy: torch.Tensor, g_logprob: Optional[torch.Tensor],
                                g_entropy: Optional[torch.Tensor], ignore_index: int) -> torch.Tensor:
    _check(logits, targets, 0)
    f32, dev = torch.float32, logits.device
    stats = check_operand("stats", stats, (*targets.shape, 2), f32, dev)
    entropy = check_operand("entropy", entropy, targets.shape, f32, dev)
    g_logprob, g_entropy = (None if g is None else check_operand(name, g, targets.shape, f32, dev)
                            for name, g in (("g_logprob", g_logprob), ("g_entropy", g_entropy)))
    return _backward(logits, targets, stats, entropy, g_logprob, g_entropy, ignore_index)


@_token_logprobs_backward_op.register_fake
def _(logits, targets, stats, entropy, g_logprob, g_entropy, ignore_index):
    return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)


def _setup_context(ctx, inputs, output) -> None:
    logits, targets, _, ignore_index = inputs
    _, entropy, stats, top_logprob, top_index = output
    ctx.save_for_backward(logits, targets, stats, entropy)
    ctx.ignore_index = ignore_index
    ctx.mark_non_differentiable(stats, top_logprob, top_index)


def _op_backward(ctx, g_logprob, g_entropy, _g_stats, _g_top, _g_index):
    logits, targets, stats, entropy = ctx.saved_tensors
    d = torch.ops.tensorcore_gemm.token_logprobs_backward(logits, targets, stats, entropy, g_logprob, g_entropy,
                                                          ctx.ignore_index)
    return d, None, None, None


_token_logprobs_op.register_autograd(_op_backward, setup_context=_setup_context)
