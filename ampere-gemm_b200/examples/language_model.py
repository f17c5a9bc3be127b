"""A small language model on this package's operators, trained and then served.

Layers of the model are  h = h + gated_ffn(layer_norm(h)), the head is
`torch.ops.tensorcore_gemm.mm`, the loss the mean of -token_logprobs with a
small entropy bonus.  There is no attention: the next token depends on the
last one only, which is what the synthetic text (a random walk on a fixed
graph of tokens) asks for.  Weights are kept in fp32 and used in fp16.

    python ampere-gemm_b200/examples/language_model.py [--steps 60] [--dim 256]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from tensorcore_gemm.ffn import gated_ffn  # noqa: E402
from tensorcore_gemm.logprobs import token_logprobs  # noqa: E402
from tensorcore_gemm.norm import layer_norm  # noqa: E402

PAD = -100


class Model:
    def __init__(self, vocab: int, dim: int, hidden: int, layers: int, device, seed: int = 0) -> None:
        gen = torch.Generator().manual_seed(seed)

        def weight(*shape, std):
            return (std * torch.randn(shape, generator=gen)).to(device).requires_grad_()

        def ones():
            return torch.ones(dim, device=device, requires_grad=True)

        self.embed = weight(vocab, dim, std=1.0)
        self.layers = [
            {"norm": ones(), "bias": torch.zeros(dim, device=device, requires_grad=True),
             "w_in": weight(2 * hidden, dim, std=dim ** -0.5), "w_out": weight(dim, hidden, std=hidden ** -0.5)}
            for _ in range(layers)
        ]
        self.norm = ones()
        self.head = weight(dim, vocab, std=dim ** -0.5)

    def parameters(self):
        return [self.embed, self.norm, self.head, *(p for layer in self.layers for p in layer.values())]

    def logits(self, tokens: torch.Tensor) -> torch.Tensor:
        """Logits of the token after each of `tokens` (any number, one included)."""
        h = self.embed[tokens].half()
        for layer in self.layers:
            y = layer_norm(h, layer["norm"], layer["bias"])
            h = h + gated_ffn(y, layer["w_in"].half(), layer["w_out"].half(), activation="silu")
        return torch.ops.tensorcore_gemm.mm(layer_norm(h, self.norm), self.head.half())


def walk(graph: torch.Tensor, length: int, gen: torch.Generator) -> torch.Tensor:
    """A text: each token is followed by one of its graph's successors."""
    pick = torch.randint(0, graph.shape[1], (length,), generator=gen).tolist()
    text = [0]
    for i in range(length):
        text.append(int(graph[text[-1], pick[i]]))
    return torch.tensor(text)


def train(model: Model, graph: torch.Tensor, steps: int, length: int, device, lr: float = 3e-3) -> list[float]:
    """Adam on -logprob - 0.01 entropy; returns the loss of each step."""
    gen = torch.Generator().manual_seed(1)
    opt = torch.optim.Adam(model.parameters(), lr=lr)
    losses = []
    for _ in range(steps):
        text = walk(graph, length, gen)
        targets = text[1:].clone()
        targets[::50] = PAD                        # padding: no loss there
        r = token_logprobs(model.logits(text[:-1].to(device)), targets.to(device), ignore_index=PAD)
        loss = -r.logprobs.sum() / (targets != PAD).sum() - 0.01 * r.entropy.mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(float(-r.logprobs.detach().sum() / (targets != PAD).sum()))
    return losses


@torch.no_grad()
def serve(model: Model, token: int, steps: int, top: int, device):
    """Greedy continuation of `token`, one token at a time, with the alternatives of every step."""
    out = []
    for _ in range(steps):
        at = torch.tensor([token], device=device)
        logits = model.logits(at)
        r = token_logprobs(logits, logits.argmax(-1), top_k=top)
        token = int(r.top_indices[0, 0])
        out.append((token, r.top_indices[0].tolist(), r.top_logprobs[0].exp().tolist(), float(r.entropy[0])))
    return out


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--vocab", type=int, default=1000)
    ap.add_argument("--dim", type=int, default=256)
    ap.add_argument("--hidden", type=int, default=688)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--length", type=int, default=2048)
    a = ap.parse_args()
    device = torch.device("cuda:0")
    graph = torch.randint(0, a.vocab, (a.vocab, 4), generator=torch.Generator().manual_seed(2))
    model = Model(a.vocab, a.dim, a.hidden, a.layers, device)
    losses = train(model, graph, a.steps, a.length, device)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} (a uniform choice among 4 successors: 1.386)")
    for token, top, p, entropy in serve(model, 0, 5, 5, device):
        print(f"token {token}: " + ", ".join(f"{t} {q:.2f}" for t, q in zip(top, p)) + f"; entropy {entropy:.2f}")


if __name__ == "__main__":
    main()
