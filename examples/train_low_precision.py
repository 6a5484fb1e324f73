"""A small language model trained and served in low precision, end to end.

    python examples/train_low_precision.py [--steps 60]

* hidden matrices: ``BlockLinear`` (FP8 products, stochastically rounded gradients),
  updated by ``MuonSR`` with FP8 momentum;
* embedding, head and norms: updated by ``AdamWReferenceSR`` with FP8 + BF16 states;
* afterwards the same layers answer token by token with their weights kept in FP8
  blocks (``quantized()`` and ``block_linear``).

The data are synthetic: sequences that walk a fixed random permutation of the
vocabulary with a few random jumps, so the loss has something to learn.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
import torch.nn.functional as F

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT / "stochastic-rounding-pytorch_b200"))

import sr_states  # noqa: E402

VOCAB, WIDTH, HIDDEN, LAYERS = 512, 256, 640, 2


class Block(torch.nn.Module):
    """A gated residual layer on the previous and the current position."""

    def __init__(self, seed, device):
        super().__init__()
        linear = sr_states.BlockLinear
        self.norm = torch.nn.Parameter(torch.ones(WIDTH, device=device, dtype=torch.bfloat16))
        self.mix = linear(2 * WIDTH, WIDTH, seed=seed, device=device)
        self.up = linear(WIDTH, HIDDEN, seed=seed + 1, device=device)
        self.down = linear(HIDDEN, WIDTH, seed=seed + 2, device=device)

    def forward(self, x, product=None):
        """``product(layer, input)`` replaces the layers' own forward when serving."""
        product = product or (lambda layer, value: layer(value))
        before = F.pad(x, (0, 0, 1, 0))[..., :-1, :]
        h = F.rms_norm(torch.cat((before, x), -1), (2 * WIDTH,))
        h = product(self.mix, h) * self.norm
        return x + product(self.down, F.silu(product(self.up, h)))


class Model(torch.nn.Module):
    def __init__(self, device):
        super().__init__()
        make = lambda *s: torch.nn.Parameter(  # noqa: E731
            (torch.randn(s, device=device) * 0.02).to(torch.bfloat16))
        self.embed, self.head = make(VOCAB, WIDTH), make(VOCAB, WIDTH)
        self.blocks = torch.nn.ModuleList(Block(10 * i, device) for i in range(LAYERS))

    def forward(self, tokens, product=None):
        x = F.embedding(tokens, self.embed)
        for block in self.blocks:
            x = block(x, product)
        return F.rms_norm(x, (WIDTH,)) @ self.head.t()

    def optimizers(self):
        hidden = [m.weight for m in self.modules() if isinstance(m, sr_states.BlockLinear)]
        other = [p for p in self.parameters() if all(p is not h for h in hidden)]
        e4m3 = sr_states.StateFormat(torch.float8_e4m3fn)
        return (sr_states.MuonSR(hidden, lr=0.02, weight_decay=0.01, state_format=e4m3, seed=1),
                sr_states.AdamWReferenceSR(other, lr=3e-3, seed=2, state_format={
                    "exp_avg": e4m3, "exp_avg_sq": sr_states.StateFormat(torch.bfloat16)}))


def batch(step, device, sequences=32, length=64):
    gen = torch.Generator().manual_seed(step)
    walk = torch.randperm(VOCAB, generator=torch.Generator().manual_seed(12345))
    tokens = torch.empty(sequences, length + 1, dtype=torch.long)
    tokens[:, 0] = torch.randint(0, VOCAB, (sequences,), generator=gen)
    for t in range(length):
        jump = torch.rand(sequences, generator=gen) < 0.05
        anywhere = torch.randint(0, VOCAB, (sequences,), generator=gen)
        tokens[:, t + 1] = torch.where(jump, anywhere, walk[tokens[:, t]])
    return tokens.to(device)


def train(steps, device):
    torch.manual_seed(0)
    model = Model(device)
    optimizers = model.optimizers()
    losses = []
    for step in range(steps):
        tokens = batch(step, device)
        logits = model(tokens[:, :-1])
        loss = F.cross_entropy(logits.float().view(-1, VOCAB), tokens[:, 1:].reshape(-1))
        loss.backward()
        for optimizer in optimizers:
            optimizer.step()
            optimizer.zero_grad()
        losses.append(loss.detach())
    return model, torch.stack(losses).tolist()


@torch.no_grad()
def serve(model, tokens, count):
    """Greedy continuation of one sequence, weights held in FP8 blocks."""
    kept = {m: m.quantized() for m in model.modules() if isinstance(m, sr_states.BlockLinear)}
    product = lambda layer, value: sr_states.block_linear(value, kept[layer])  # noqa: E731
    for _ in range(count):
        # the layers look one position back: LAYERS + 1 positions decide the next token
        logits = model(tokens[:, -(LAYERS + 1):], product)
        tokens = torch.cat((tokens, logits[:, -1:].float().argmax(-1)), 1)
    return tokens


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=60)
    args = parser.parse_args()
    device = torch.device("cuda", torch.cuda.current_device())
    model, losses = train(args.steps, device)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} in {args.steps} steps")
    start = batch(10**6, device)[:1, :4]
    print("continued:", serve(model, start, 12)[0].tolist())


if __name__ == "__main__":
    main()
