"""Fine-tune a block-pruned feed-forward block back to its dense teacher.

The student keeps a share of the teacher's up-projection (32x32 blocks of the
largest norm, a SparseLinear) and is trained on the teacher's top logits:

    h = x + down(gelu(up(norm(x)))),  logits = head(norm(h))

with layer_norm, SparseLinear, fused_linear (the down-projection adds the
residual in its epilogue) and distillation_loss.  Run on an MI355X:

    python examples/distill_pruned.py --steps 100
"""

from __future__ import annotations

import argparse
import copy
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import void_amd  # noqa: E402


class Teacher(torch.nn.Module):
    """The dense block, random weights."""

    def __init__(self, width: int, hidden: int, vocab: int, dtype: torch.dtype):
        super().__init__()
        self.norm = void_amd.LayerNorm(width, dtype=dtype)
        self.up = void_amd.FusedLinear(width, hidden, "gelu", dtype=dtype)
        self.down = void_amd.FusedLinear(hidden, width, dtype=dtype)
        self.last = void_amd.LayerNorm(width, dtype=dtype)
        self.head = void_amd.FusedLinear(width, vocab, bias=False, dtype=dtype)
        torch.nn.init.normal_(self.up.weight, std=2 * width ** -0.5)
        torch.nn.init.normal_(self.head.weight, std=2 * width ** -0.5)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.head(self.last(self.down(self.up(self.norm(x)), x)))


def prune(weight: torch.Tensor, keep: float) -> "void_amd.VOIDTensor":
    """The weight's 32x32 blocks of the largest norm as a VOID tensor."""
    M, K = weight.shape
    blocks = weight.float().view(M // 32, 32, K // 32, 32)
    norm = blocks.square().sum((1, 3))
    floor = norm.flatten().kthvalue(max(1, int(norm.numel() * (1 - keep)))).values
    kept = (blocks * (norm > floor)[:, None, :, None]).reshape(M, K)
    return void_amd.dense_to_void(kept.cpu()).to_dtype(weight.dtype)


class Student(torch.nn.Module):
    """The teacher with a sparse up-projection."""

    def __init__(self, teacher: Teacher, keep: float):
        super().__init__()
        self.norm, self.down, self.last, self.head = teacher.norm, teacher.down, teacher.last, teacher.head
        self.up = void_amd.SparseLinear(teacher.up.in_features, teacher.up.out_features,
                                        prune(teacher.up.weight.detach(), keep))
        with torch.no_grad():
            self.up.bias.copy_(teacher.up.bias)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        y = torch.nn.functional.gelu(self.up(self.norm(x)), approximate="tanh")
        return self.head(self.last(self.down(y, x)))


def train(steps: int = 50, tokens: int = 512, width: int = 512, hidden: int = 1024, vocab: int = 4096, k: int = 32,
          keep: float = 0.25, temperature: float = 2.0, lr: float = 1e-3, dtype: torch.dtype = torch.bfloat16,
          device: str = "cuda", seed: int = 0, report=print) -> list:
    """The steps' losses above the teacher's own: a student equal to the teacher still
    spreads some probability outside the k entries, which the loss counts."""
    torch.manual_seed(seed)
    teacher = Teacher(width, hidden, vocab, dtype).to(device)
    student = Student(copy.deepcopy(teacher), keep).to(device)
    optimiser = torch.optim.AdamW(student.parameters(), lr=lr, weight_decay=0.0)
    losses = []
    for step in range(steps):
        x = torch.randn(tokens, width, device=device).to(dtype)
        with torch.no_grad():
            goal = teacher(x)
            top, index = goal.topk(k, dim=-1)
            index[:tokens // 8] = -1  # prompt tokens: no loss
            least = void_amd.distillation_loss(goal, top, index, temperature=temperature)
        loss = void_amd.distillation_loss(student(x), top, index, temperature=temperature)
        optimiser.zero_grad(set_to_none=True)
        loss.backward()
        optimiser.step()
        losses.append(loss.detach() - least)
        if report and step % 10 == 0:
            report(f"step {step:4d}  loss {float(loss.detach()):.4f}, {float(losses[-1]):.4f} above the teacher's")
    losses = [float(x) for x in losses]
    if report:
        report(f"above the teacher's: {losses[0]:.4f} -> {losses[-1]:.4f}")
    return losses


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--steps", type=int, default=50)
    parser.add_argument("--tokens", type=int, default=512)
    parser.add_argument("--keep", type=float, default=0.25, help="share of the up-projection's blocks that stay")
    args = parser.parse_args()
    train(steps=args.steps, tokens=args.tokens, keep=args.keep)
