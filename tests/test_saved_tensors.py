"""The dense operators' backward passes read what autograd gives back, wherever
that lies: saved-tensor hooks and checkpoints return other tensors than the
forward pass had, whose own memory is free by then.

On the CPU the library is replaced by a recorder of the addresses it is given.
On the GPU every gradient has the bits of the plain call: nothing is computed
differently.
"""

import ctypes

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import void_amd
from void_amd import _lib, _runtime, distill

gpu_only = pytest.mark.gpu


class Recorder:
    """In the library's place: the calls of each entry, sizes of 0, status OK."""

    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        if name.startswith("__"):
            raise AttributeError(name)

        def entry(*args):
            # A structure is read while its call runs.
            args = [type(a._obj).from_buffer_copy(a._obj) if hasattr(a, "_obj") else a for a in args]
            self.calls.setdefault(name, []).append(args)
            return 1 if name == "void_distill_slices" else 0
        return entry


@pytest.fixture
def recorder(monkeypatch):
    r = Recorder()
    monkeypatch.setattr(_lib, "lib", lambda: r)
    monkeypatch.setattr(_runtime, "require_gpu", lambda t, what: None)
    monkeypatch.setattr(distill, "raw_stream", lambda device: 0)
    return r


class Moved:
    """Hooks that keep a copy of what is saved and hand out another one, in a layout of `lay`'s making."""

    def __init__(self, lay=torch.clone):
        self.given, self.lay = [], lay

    def pack(self, t):
        return t.detach().clone()

    def unpack(self, t):
        t = self.lay(t)
        self.given.append(t)
        return t

    def __call__(self):
        return torch.autograd.graph.saved_tensors_hooks(self.pack, self.unpack)


def distill_inputs(device, R=6, V=200, k=5, dtype=torch.float32):
    g = torch.Generator().manual_seed(R + V)
    s = torch.randn(R, V, generator=g) * 2
    idx = torch.rand(R, V, generator=g).argsort(1)[:, :k]
    t = torch.randn(R, k, generator=g) * 2 + 5
    idx[1] = -1
    return s.to(device, dtype), t.to(device, dtype), idx.to(device)


def test_distillation_backward_reads_the_unpacked_tensors(recorder):
    s, t, idx = distill_inputs("cpu")
    # Rows of another pitch in the forward pass: the strides are the unpacked tensors' too.
    s = torch.cat((s, s), 1)[:, :200].requires_grad_()
    hooks = Moved()
    with hooks():
        loss = void_amd.distillation_loss(s, t, idx)
    torch.autograd.grad(loss, s)
    (before, *_), = recorder.calls["void_distill_loss"]
    (args, parts, *_), = recorder.calls["void_distill_grad"]
    at = {u.data_ptr(): u for u in hooks.given}
    assert before.logits == s.data_ptr() and before.ld == 400
    for pointer, shape in ((args.logits, (6, 200)), (args.teacher, (6, 5)), (args.index, (6, 5)), (parts, (6, 1, 2))):
        assert at[pointer].shape == shape
    assert (args.ld, args.ldt, args.ldi) == (at[args.logits].stride(0), at[args.teacher].stride(0), at[args.index].stride(0))
    assert (args.rows, args.vocab, args.k, args.dtype, args.index_bytes) == (6, 200, 5, 0, 8)


def overwritten(device):
    """Takes and fills the memory that was freed, so that a stale address reads something else."""
    for n in (1 << 10, 1 << 14, 1 << 18, 1 << 22):
        for _ in range(8):
            torch.full((n,), float("nan"), device=device)


@gpu_only
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V", [(600, 3000), (3, 20001)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_distillation_under_hooks_and_checkpoints(gpu, dtype, R, V, reduction):
    x, t, idx = distill_inputs(gpu, R, V, dtype=dtype)

    def loss(head):
        # The logits are made here, and freed with what the hooks or the checkpoint drop.
        return void_amd.distillation_loss(head * 1.5, t * 1.0, idx + 0, 2.0, reduction).sum()

    def gradient(around):
        leaf = x.detach().requires_grad_()
        out = around(leaf)
        overwritten(gpu)
        out.backward()
        return leaf.grad

    want = gradient(loss)
    assert torch.isfinite(want).all() and want.any()

    def hooked(ctx):
        def run(leaf):
            with ctx():
                return loss(leaf)
        return run
    for around in (hooked(Moved()), hooked(torch.autograd.graph.save_on_cpu),
                   lambda leaf: checkpoint(loss, leaf, use_reentrant=False),
                   lambda leaf: checkpoint(loss, leaf, use_reentrant=True)):
        assert torch.equal(gradient(around), want)
