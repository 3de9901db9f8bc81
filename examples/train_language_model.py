"""Train a small mixture-of-experts language model with ApexW and the operators around the step.

    python examples/train_language_model.py [--steps 60]

The model predicts a token from the two before it: an embedding of each, scaled, residual blocks of a layer norm, a
router that sends each token to two experts and two expert products with a GELU between them, and a head that shares the
embedding's table.  Sequences are of different lengths; their padding has the id -1, which the embedding and the loss
leave out, and goes to no expert.  The logits are never stored, and nothing is read back on the host within a step.  The
parameters are bf16; gradients of two micro-batches are accumulated in fp32 and clipped by their global norm into the
parameters' type, then ApexW steps.
"""

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch

import apexw_amd


class Block(torch.nn.Module):
    def __init__(self, width, hidden, experts, choices):
        super().__init__()
        self.choices = choices
        self.norm_weight = torch.nn.Parameter(torch.ones(width))
        self.norm_bias = torch.nn.Parameter(torch.zeros(width))
        self.router = torch.nn.Parameter(torch.randn(experts, width) * width ** -0.5)
        self.up = torch.nn.Parameter(torch.randn(experts, hidden, width) * width ** -0.5)
        self.down = torch.nn.Parameter(torch.randn(experts, width, hidden) * hidden ** -0.5)

    def forward(self, x, padding):
        h = apexw_amd.layer_norm(x, self.norm_weight, self.norm_bias)
        scores, expert = torch.topk((h @ self.router.t()).float(), self.choices)
        order = apexw_amd.expert_order(torch.where(padding[:, None], -1, expert), self.router.shape[0])
        y = apexw_amd.expert_dispatch(h, order)
        y = apexw_amd.expert_matmul(y, self.up, order.ends)
        y = apexw_amd.expert_matmul(torch.nn.functional.gelu(y), self.down, order.ends)
        return x + apexw_amd.expert_combine(y, order, torch.softmax(scores, dim=-1))


class LanguageModel(torch.nn.Module):
    def __init__(self, vocab, width, hidden, experts, choices=2, layers=2):
        super().__init__()
        self.table = torch.nn.Parameter(torch.randn(vocab, width) * width ** -0.5)
        self.before = torch.nn.Parameter(torch.randn(vocab, width) * width ** -0.5)
        self.blocks = torch.nn.ModuleList(Block(width, hidden, experts, choices) for _ in range(layers))
        self.norm_weight = torch.nn.Parameter(torch.ones(width))
        self.norm_bias = torch.nn.Parameter(torch.zeros(width))

    def forward(self, ids, target, reduction="mean"):
        """The loss of predicting `target` from `ids`, (sequences, length) each, -1 for padding."""
        scale = self.table.shape[1] ** 0.5
        before = torch.nn.functional.pad(ids[:, :-1], (1, 0), value=-1)
        x = apexw_amd.embedding(ids, self.table, scale) + apexw_amd.embedding(before, self.before, scale)
        x, padding = x.flatten(0, 1), ids.flatten() < 0
        for block in self.blocks:
            x = block(x, padding)
        h = apexw_amd.layer_norm(x, self.norm_weight, self.norm_bias)
        return apexw_amd.linear_cross_entropy(h, self.table, target.flatten(), ignore_index=-1, reduction=reduction)


def batch(table, sequences, length, generator):
    """Sequences in which each token follows from the one before by a fixed table, one time in eight by chance."""
    vocab, device = table.shape[0], table.device
    ids = torch.empty(sequences, length + 1, dtype=torch.int64, device=device)
    ids[:, 0] = torch.randint(0, vocab, (sequences,), generator=generator, device=device)
    for t in range(length):
        chance = torch.randint(0, vocab, (sequences,), generator=generator, device=device)
        ids[:, t + 1] = torch.where(torch.rand(sequences, generator=generator, device=device) < 0.125, chance, table[ids[:, t]])
    lengths = torch.randint(length // 2, length + 1, (sequences, 1), generator=generator, device=device)
    here = torch.arange(length, device=device) < lengths
    return torch.where(here, ids[:, :-1], -1), torch.where(here, ids[:, 1:], -1)


def train(steps=60, vocab=2000, width=128, hidden=256, experts=8, sequences=32, length=64, micro=2, max_norm=0.5, seed=0):
    """The losses of the steps, and the gradient norms before the clip."""
    torch.manual_seed(seed)
    device = torch.device("cuda")
    generator = torch.Generator(device=device).manual_seed(seed)
    model = LanguageModel(vocab, width, hidden, experts).to(device=device, dtype=torch.bfloat16)
    follows = torch.randint(0, vocab, (vocab,), generator=generator, device=device)
    params = list(model.parameters())
    opt = apexw_amd.ApexW(params, lr=4e-3, weight_decay=0.01, adamw_compat=True)
    main = [torch.zeros(p.shape, dtype=torch.float32, device=device) for p in params]
    losses, norms = [], []
    for _ in range(steps):
        for g in main:
            g.zero_()
        total = torch.zeros((), device=device)
        for _ in range(micro):
            loss = model(*batch(follows, sequences, length, generator))
            for g, d in zip(main, torch.autograd.grad(loss / micro, params)):
                g += d
            total += loss.detach() / micro
        for p in params:
            if p.grad is None:
                p.grad = torch.empty_like(p)
        norms.append(apexw_amd.clip_grads(main, max_norm, out=[p.grad for p in params]))
        opt.step()
        losses.append(total)
    return torch.stack(losses).tolist(), torch.stack(norms).tolist()


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--steps", type=int, default=60)
    args = parser.parse_args()
    losses, norms = train(args.steps)
    for i in range(0, len(losses), max(1, len(losses) // 10)):
        print(f"step {i:4d}  loss {losses[i]:.4f}  gradient norm {norms[i]:.3f}")
    print(f"last loss {losses[-1]:.4f}")
