"""Train a small hybrid language model and decode from it, on one GPU.

    python examples/train_hybrid_lm.py [--steps N] [--nested]

The model's layers mix tokens by gated linear recurrences (``--nested`` makes
every other layer a nested GDN-2 layer); its embedding, recurrences and weight
updates run on this package's kernels: the scaled lookup with its gradient,
the scan with its backward and the one-token step, and Muon's orthogonalised
updates. The data are synthetic: token frequencies fall as 1 / rank, and three
times out of four a token is followed by its own fixed successor.
"""

from __future__ import annotations

import argparse
import pathlib
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1]))

from nested_recurrent_memory_b200 import check_status  # noqa: E402
from nested_recurrent_memory_b200.model import ModelConfig, NestedGDN2ForCausalLM  # noqa: E402
from nested_recurrent_memory_b200.optim import Muon, split_parameters  # noqa: E402


def batch(gen, B, T, vocab):
    """[B, T] token ids: a random token, or the fixed successor of the last one."""
    fresh = (((vocab + 1.0) ** torch.rand(B, T, generator=gen)).long() - 1).clamp_(0, vocab - 1)
    follow = torch.rand(B, T, generator=gen) < 0.75
    for t in range(1, T):
        fresh[:, t] = torch.where(follow[:, t], successor(fresh[:, t - 1], vocab), fresh[:, t])
    return fresh.cuda()


def successor(ids, vocab):
    return (ids * 5 + 3) % vocab


def train(steps=30, nested=False, B=8, T=256, vocab=512, layers=2, seed=0, log=print):
    torch.manual_seed(seed)
    gen = torch.Generator().manual_seed(seed)
    cfg = ModelConfig(vocab_size=vocab, hidden_size=256, num_hidden_layers=layers, num_heads=2,
                      head_dim=128, num_levels=3, firing_intervals=(1, 2, 4),
                      n_queries_per_level=(64, 64), embed_scale=16.0,
                      recurrent_layers=tuple(range(0, layers, 2) if nested else range(layers)))
    model = NestedGDN2ForCausalLM(cfg).cuda()
    matrices, rest = split_parameters(model)
    optimisers = [Muon(matrices, lr=0.02), torch.optim.AdamW(rest, lr=3e-3, weight_decay=0.0)]
    losses = []
    for i in range(steps):
        ids = batch(gen, B, T + 1, vocab)
        loss = F.cross_entropy(model(ids[:, :-1]).flatten(0, 1), ids[:, 1:].flatten())
        loss.backward()
        for opt in optimisers:
            opt.step()
            opt.zero_grad(set_to_none=True)
        loss = loss.detach()
        losses.append(loss)
        if log and (i % 10 == 0 or i + 1 == steps):
            log(f"step {i}: loss {float(loss):.4f}")
    check_status()
    return model, [float(x) for x in losses]


@torch.no_grad()
def decode(model, prompt, n):
    """Greedy continuation of [B, T] prompt ids by n tokens."""
    logits, states = model.prefill(prompt)
    ids, out = logits[:, -1].argmax(-1), []
    for _ in range(n):
        out.append(ids)
        ids = model.step(ids, states).argmax(-1)
    return torch.stack(out, 1)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=100)
    ap.add_argument("--nested", action="store_true")
    args = ap.parse_args()
    model, losses = train(args.steps, args.nested)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f}")
    if not args.nested:
        ids = batch(torch.Generator().manual_seed(99), 2, 32, 512)
        out = torch.cat([ids[:, -1:], decode(model, ids, 8)], 1)
        print("continuation", out[0].tolist())
        print("successors  ", successor(out[0], 512).tolist()[:-1])


if __name__ == "__main__":
    main()
