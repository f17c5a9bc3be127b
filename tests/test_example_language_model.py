"""The example model: its operators together, trained and served."""
from __future__ import annotations

import importlib.util
import math
from pathlib import Path

import pytest
import torch

PATH = Path(__file__).resolve().parent.parent / "ampere-gemm_b200" / "examples" / "language_model.py"


def load():
    spec = importlib.util.spec_from_file_location("language_model_example", PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_text_follows_the_graph():
    ex = load()
    graph = torch.randint(0, 50, (50, 4), generator=torch.Generator().manual_seed(0))
    text = ex.walk(graph, 200, torch.Generator().manual_seed(1))
    assert all(int(b) in graph[int(a)].tolist() for a, b in zip(text, text[1:]))


@pytest.mark.gpu
def test_gradients_match_plain_torch(cuda_device, native_lib):
    """One step's loss and gradients against the same model in 64-bit torch operations.

    Activations, weights and the gradients between layers are rounded to 11
    bits at each of about ten steps along a path; 3 % of a gradient's norm
    allows for that and for their amplification by the norms."""
    ex = load()
    model = ex.Model(300, 64, 136, 2, cuda_device)
    text = torch.randint(0, 300, (97,), generator=torch.Generator().manual_seed(3)).to(cuda_device)
    targets = text[1:].clone()
    targets[5] = ex.PAD
    r = ex.token_logprobs(model.logits(text[:-1]), targets, ignore_index=ex.PAD)
    loss = -r.logprobs.sum() / 95 - 0.01 * r.entropy.mean()
    grads = torch.autograd.grad(loss, model.parameters())

    params = [p.detach().double().requires_grad_() for p in model.parameters()]
    embed, norm, head, *rest = params
    h = embed[text[:-1]]
    for i in range(2):
        w, b, w_in, w_out = rest[4 * i:4 * i + 4]
        g, u = (torch.nn.functional.layer_norm(h, (64,), w, b) @ w_in.t()).chunk(2, -1)
        h = h + (torch.nn.functional.silu(g) * u) @ w_out.t()
    lp = torch.log_softmax(torch.nn.functional.layer_norm(h, (64,), norm) @ head, -1)
    given = targets != ex.PAD
    picked = lp.gather(1, targets.clamp(min=0)[:, None])[:, 0][given]
    ref = -picked.sum() / 95 + 0.01 * (lp.exp() * lp).sum(-1).mean()
    assert abs(float(loss.detach()) - float(ref.detach())) < 0.01 * abs(float(ref.detach()))
    for got, want in zip(grads, torch.autograd.grad(ref, params)):
        assert (got.double() - want).norm() <= 0.03 * want.norm() + 1e-6


@pytest.mark.gpu
def test_training_learns_and_serving_follows(cuda_device, native_lib):
    ex = load()
    graph = torch.randint(0, 200, (200, 4), generator=torch.Generator().manual_seed(2))
    model = ex.Model(200, 128, 344, 2, cuda_device)
    losses = ex.train(model, graph, 60, 1024, cuda_device)
    assert losses[0] > 4.0 and all(math.isfinite(v) for v in losses)
    assert losses[-1] < 2.0                      # ln 4 = 1.39 is the text's own entropy
    token = 0
    for nxt, top, p, _ in ex.serve(model, 0, 6, 4, cuda_device):
        assert nxt in graph[token].tolist()
        assert sum(p) > 0.5 and top[0] == nxt
        token = nxt
