"""A model of words whose tokens run through hyper-connected blocks: trained, scored and run word by word.

The two ends of the network share one table: ``embedding`` looks a token's row up, scales it and copies it
into the residual streams; the streams' normalised mean meets the same table in ``linear_cross_entropy``,
which never keeps the logits.  Between them run the blocks of ``hyper_block.py``.  Blocks mix the streams
of each token by itself, so what is learnt is which word follows which.

    PYTHONPATH=flash-hyperconnections_amd python examples/word_model.py [--device cuda] [--steps 60]

The 16-bit types need the GPU: native matrix exponentials of them on the CPU are NaN.
"""

import argparse
import importlib.util
from pathlib import Path

import torch

import flash_hypercons as fh

_spec = importlib.util.spec_from_file_location("hyper_block", Path(__file__).with_name("hyper_block.py"))
hyper_block = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(hyper_block)

PADDING = 0  # a word that stands for none: no gradient in the table, and no target


class WordModel(torch.nn.Module):
    def __init__(self, words=1000, width=64, streams=4, depth=2, device="cpu", dtype=torch.float32):
        super().__init__()
        self.streams, self.scale = streams, width**0.5
        self.table = torch.nn.Parameter((torch.randn(words, width) * width**-0.5).to(device, dtype))
        self.blocks = torch.nn.ModuleList(hyper_block.Block(width, streams, device, dtype) for _ in range(depth))
        self.norm = torch.nn.Parameter(torch.ones(width, device=device, dtype=dtype))

    def hidden(self, tokens: torch.Tensor) -> torch.Tensor:
        """[tokens, width]: what each token says of the next one."""
        streams = fh.embedding(tokens, self.table, scale=self.scale, streams=self.streams, padding_idx=PADDING)
        for block in self.blocks:
            streams = block(streams)
        return fh.layer_norm(streams.mean(1), self.norm)

    def forward(self, tokens: torch.Tensor, targets: torch.Tensor, reduction: str = "mean") -> torch.Tensor:
        return fh.linear_cross_entropy(self.hidden(tokens), self.table, targets, ignore_index=PADDING,
                                       reduction=reduction)


def sequences(words: int, count: int, length: int, gen: torch.Generator):
    """Words that follow each other by a fixed rule half of the time; ends of sequences are padding."""
    words_in = torch.randint(1, words, (count, length + 1), generator=gen)
    for i in range(length):
        rule = (words_in[:, i] * 7 + 3) % (words - 1) + 1
        words_in[:, i + 1] = torch.where(torch.rand(count, generator=gen) < 0.5, rule, words_in[:, i + 1])
    ends = torch.randint(length // 2, length + 2, (count, 1), generator=gen)
    words_in[torch.arange(length + 1) >= ends] = PADDING
    return words_in[:, :-1].reshape(-1), words_in[:, 1:].reshape(-1)


def train(model: WordModel, steps: int, count: int = 64, length: int = 32, rate: float = 0.5, seed: int = 0):
    """Losses and the gradients' norms before clipping."""
    gen = torch.Generator().manual_seed(seed)
    device, words = model.table.device, model.table.shape[0]
    masters = [p.detach().float() for p in model.parameters()]  # 16-bit parameters would lose small updates
    losses, norms = [], []
    for _ in range(steps):
        tokens, targets = (t.to(device) for t in sequences(words, count, length, gen))
        loss = model(tokens, targets)
        model.zero_grad()
        loss.backward()
        norms.append(fh.clip_grad_norm_(model.parameters(), 1.0))
        with torch.no_grad():
            for p, master in zip(model.parameters(), masters):
                p.copy_(master.sub_(rate * p.grad.float()))
        losses.append(loss.detach())
    return [v.item() for v in losses], [v.item() for v in norms]


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    ap.add_argument("--dtype", default="float32", choices=("float32", "bfloat16", "float16"))
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--words", type=int, default=1000)
    args = ap.parse_args()
    torch.manual_seed(0)
    model = WordModel(args.words, device=args.device, dtype=getattr(torch, args.dtype))
    losses, norms = train(model, args.steps)
    for i in range(0, args.steps, max(1, args.steps // 6)):
        print(f"step {i:4d}  loss {losses[i]:.4f}  gradient norm {norms[i]:.3f}")
    with torch.no_grad():  # scoring: each position by itself, then one token at a time
        tokens, targets = (t.to(args.device) for t in sequences(args.words, 2, 16, torch.Generator().manual_seed(1)))
        together = model(tokens, targets, "none")
        alone = torch.cat([model(t.view(1), n.view(1), "none") for t, n in zip(tokens, targets)])
        print(f"negative log-probability a word {together[targets != PADDING].mean().item():.4f}")
        print(f"token by token against together: {(together - alone).abs().max().item():.1e}")


if __name__ == "__main__":
    main()
