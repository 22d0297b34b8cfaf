"""A stack of hyper-connected feed-forward blocks: trained, then run token by token.

Each block mixes the n residual streams of every token by ``exp(h)`` (``mix_streams``), where h comes
from the token's normalised streams (``layer_norm``, ``linear``), and feeds the first stream through
``layer_norm`` and two ``linear`` layers, the activation and the residual in their epilogues.  The
gradients are clipped by their global norm (``clip_grad_norm_``).

    PYTHONPATH=flash-hyperconnections_amd python examples/hyper_block.py [--device cuda] [--steps 60]

The 16-bit types need the GPU: native matrix exponentials of them on the CPU are NaN.
"""

import argparse

import torch

import flash_hypercons as fh


class Block(torch.nn.Module):
    """One mixing of [tokens, streams, width] and the feed-forward block on the first stream."""

    def __init__(self, width: int, streams: int, device, dtype):
        super().__init__()
        self.streams = streams

        def normal(rows, cols, scale):
            return torch.nn.Parameter((torch.randn(rows, cols) * scale * cols**-0.5).to(device, dtype))

        def constant(value, n):
            return torch.nn.Parameter(torch.full((n,), value, device=device, dtype=dtype))

        both = streams * width
        self.mix_scale, self.mix_shift = constant(1.0, both), constant(0.0, both)
        self.generator, self.offset = normal(streams * streams, both, 0.1), constant(0.0, streams * streams)
        self.scale, self.shift = constant(1.0, width), constant(0.0, width)
        self.up, self.up_bias = normal(4 * width, width, 1.0), constant(0.0, 4 * width)
        self.down, self.down_bias = normal(width, 4 * width, 0.5), constant(0.0, width)

    def forward(self, streams: torch.Tensor) -> torch.Tensor:
        flat = fh.layer_norm(streams.flatten(1), self.mix_scale, self.mix_shift)
        h = fh.linear(flat, self.generator, self.offset).view(-1, self.streams, self.streams)
        streams = fh.mix_streams(h, streams)
        read = streams[:, 0]  # rows a stream apart, read in place
        hidden = fh.linear(fh.layer_norm(read, self.scale, self.shift), self.up, self.up_bias, activation="gelu")
        written = fh.linear(hidden, self.down, self.down_bias, residual=read)
        return torch.cat((written.unsqueeze(1), streams[:, 1:]), 1)


class Stack(torch.nn.Module):
    def __init__(self, width=64, streams=4, depth=3, device="cpu", dtype=torch.float32):
        super().__init__()
        self.streams = streams
        self.blocks = torch.nn.ModuleList(Block(width, streams, device, dtype) for _ in range(depth))

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        streams = tokens.unsqueeze(1).repeat(1, self.streams, 1)
        for block in self.blocks:
            streams = block(streams)
        return streams.float().mean(1)


def train(stack: Stack, steps: int, tokens: int = 256, rate: float = 0.05, max_norm: float = 1.0, seed: int = 0):
    """Fits a fixed random map; returns the losses and the gradients' norms before clipping."""
    first = next(stack.parameters())
    gen = torch.Generator().manual_seed(seed)
    width = stack.blocks[0].scale.numel()
    teacher = (torch.randn(width, width, generator=gen) * width**-0.5).to(first.device)
    masters = [p.detach().float() for p in stack.parameters()]  # 16-bit parameters would lose small updates
    losses, norms = [], []
    for _ in range(steps):
        x = torch.randn(tokens, width, generator=gen).to(first.device)
        loss = (stack(x.to(first.dtype)) - torch.tanh(x @ teacher)).square().mean()
        stack.zero_grad()
        loss.backward()
        norms.append(fh.clip_grad_norm_(stack.parameters(), max_norm))
        with torch.no_grad():
            for p, master in zip(stack.parameters(), masters):
                p.copy_(master.sub_(rate * p.grad.float()))
        losses.append(loss.detach())
    return [v.item() for v in losses], [v.item() for v in norms]


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    ap.add_argument("--dtype", default="float32", choices=("float32", "bfloat16", "float16"))
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--width", type=int, default=64)
    args = ap.parse_args()
    torch.manual_seed(0)
    stack = Stack(args.width, device=args.device, dtype=getattr(torch, args.dtype))
    losses, norms = train(stack, args.steps)
    for i in range(0, args.steps, max(1, args.steps // 6)):
        print(f"step {i:4d}  loss {losses[i]:.4f}  gradient norm {norms[i]:.3f}")
    print(f"last loss {losses[-1]:.4f}")
    with torch.no_grad():  # serving: the same network, one token at a time
        tokens = torch.randn(8, args.width).to(args.device, getattr(torch, args.dtype))
        together, alone = stack(tokens), torch.cat([stack(t.unsqueeze(0)) for t in tokens])
        print(f"token by token against together: {(together - alone).abs().max().item():.1e}")


if __name__ == "__main__":
    main()
