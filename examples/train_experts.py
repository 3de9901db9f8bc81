"""Train a small mixture-of-experts block with ApexW and the operators around the step.

    python examples/train_experts.py [--steps 60]

A residual block over tokens: layer norm, a router that sends each token to one expert, two expert products
with a GELU between them.  The parameters are bf16; the gradients of two micro-batches are accumulated in
fp32 and clipped by their global norm into the parameters' type, then ApexW steps.  The block learns a fixed
random map of the tokens; the loss falls by more than a quarter within the default steps.
"""

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch

import apexw_amd


class ExpertBlock(torch.nn.Module):
    def __init__(self, width, hidden, experts):
        super().__init__()
        self.norm_weight = torch.nn.Parameter(torch.ones(width))
        self.norm_bias = torch.nn.Parameter(torch.zeros(width))
        self.router = torch.nn.Parameter(torch.randn(experts, width) * width ** -0.5)
        self.up = torch.nn.Parameter(torch.randn(experts, hidden, width) * width ** -0.5)
        self.down = torch.nn.Parameter(torch.randn(experts, width, hidden) * hidden ** -0.5)

    def forward(self, x):
        h = apexw_amd.layer_norm(x, self.norm_weight, self.norm_bias)
        scores = torch.softmax((h @ self.router.t()).float(), dim=-1)
        weight, expert = scores.max(dim=-1)
        # rows sorted by expert, and one past each expert's last row: nothing leaves the device
        order = torch.argsort(expert, stable=True)
        ends = torch.bincount(expert, minlength=self.router.shape[0]).cumsum(0).to(torch.int32)
        y = apexw_amd.expert_matmul(h[order], self.up, ends)
        y = apexw_amd.expert_matmul(torch.nn.functional.gelu(y), self.down, ends)
        back = torch.empty_like(order)
        back[order] = torch.arange(len(order), device=order.device)
        return x + y[back] * weight.to(x.dtype)[:, None]


def train(steps=60, width=256, hidden=512, experts=8, tokens=1024, micro=2, max_norm=0.1, seed=0):
    """The losses of the steps, and the gradient norms before the clip."""
    torch.manual_seed(seed)
    device = torch.device("cuda")
    block = ExpertBlock(width, hidden, experts).to(device=device, dtype=torch.bfloat16)
    target = (torch.randn(width, width, device=device) * width ** -0.5).bfloat16()
    params = list(block.parameters())
    opt = apexw_amd.ApexW(params, lr=2e-3, weight_decay=0.01, adamw_compat=True)
    main = [torch.zeros(p.shape, dtype=torch.float32, device=device) for p in params]
    losses, norms = [], []
    for _ in range(steps):
        for g in main:
            g.zero_()
        total = torch.zeros((), device=device)
        for _ in range(micro):
            x = torch.randn(tokens, width, device=device, dtype=torch.bfloat16)
            loss = (block(x) - x @ target).float().square().mean()
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
