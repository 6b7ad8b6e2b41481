"""examples/distill_pruned.py: layer norm, the sparse layer, the dense layers and
the distillation loss in one training loop, whose loss falls; and one step's
gradients against the same block in 64 bits."""

import copy
import importlib.util
from pathlib import Path

import pytest
import torch

import void_amd

pytestmark = pytest.mark.gpu

PATH = Path(__file__).resolve().parents[1] / "examples" / "distill_pruned.py"


def example():
    spec = importlib.util.spec_from_file_location("distill_pruned", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_loss_falls(gpu, dtype):
    losses = example().train(steps=40, tokens=256, width=128, hidden=256, vocab=1000, k=16, dtype=dtype, report=None)
    # Above the teacher's own loss (which is not 0: its probability outside the k entries).
    assert losses[0] > 0 and sum(losses[-5:]) < 0.5 * sum(losses[:5])


def test_gradients_of_the_whole_step(gpu):
    ex = example()
    torch.manual_seed(1)
    width, hidden, vocab, k, T = 96, 160, 300, 12, 2.0
    teacher = ex.Teacher(width, hidden, vocab, torch.float32).to(gpu)
    student = ex.Student(copy.deepcopy(teacher), 0.3).to(gpu)
    x = torch.randn(80, width, device=gpu)
    with torch.no_grad():
        top, index = teacher(x).topk(k, dim=-1)
        index[:10] = -1
    void_amd.distillation_loss(student(x), top, index, temperature=T).backward()

    w = student.up.sparse_weight
    values = w.values.detach().double().requires_grad_()
    dense = torch.zeros(hidden // 32, width // 32, 32, 32, dtype=torch.float64, device=gpu)
    dense = dense.index_put((w.block_rows.long(), w.block_cols.long()), values)
    dense = dense.permute(0, 2, 1, 3).reshape(hidden, width)
    p = {n: q.detach().double().requires_grad_() for n, q in student.named_parameters()}
    norm = lambda t, name: torch.nn.functional.layer_norm(t, (width,), p[name + ".weight"], p[name + ".bias"])
    xd = x.double()
    up = torch.nn.functional.gelu(norm(xd, "norm") @ dense.t() + p["up.bias"], approximate="tanh")
    h = up @ p["down.weight"].t() + p["down.bias"] + xd
    logits = norm(h, "last") @ p["head.weight"].t()
    keep = index[:, 0] >= 0
    t = torch.softmax(top[keep].double() / T, 1)
    logq = torch.log_softmax(logits[keep] / T, 1).gather(1, index[keep])
    (T * T * (t * (t.log() - logq)).sum(1).mean()).backward()
    for name, q in student.named_parameters():
        want = values.grad if name == "up.sparse_weight.values" else p[name].grad
        # Five 32-bit products in a row, each sum of at most 300 terms: 2^-24 sqrt(300) each, 8 times that in all.
        assert (q.grad.double() - want).norm() <= 8 * 2.0 ** -24 * 300 ** 0.5 * 5 * want.norm(), name
