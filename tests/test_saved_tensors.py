"""The dense operators' backward passes read what autograd gives back, wherever
that lies: saved-tensor hooks and checkpoints return other tensors than the
forward pass had, whose own memory is free by then.

On the CPU the library is replaced by a recorder of the addresses it is given.
On the GPU every gradient has the bits of the plain call: nothing is computed
differently.
"""

import ctypes

import numpy as np
import pytest
import torch
from torch.utils.checkpoint import checkpoint

import void_amd
from void_amd import _lib, _runtime, distill, linear, norm

gpu_only = pytest.mark.gpu


class Recorder:
    """In the library's place: the calls of each entry, sizes of 0, status OK.  `look` names
    functions that look at an entry's arguments while it runs."""

    def __init__(self):
        self.calls, self.look = {}, {}

    def __getattr__(self, name):
        if name.startswith("__"):
            raise AttributeError(name)

        def entry(*args):
            # A structure is read while its call runs.
            args = [type(a._obj).from_buffer_copy(a._obj) if hasattr(a, "_obj") else a for a in args]
            self.calls.setdefault(name, []).append(args)
            if name in self.look:
                self.look[name](*args)
            return 1 if name == "void_distill_slices" else 0
        return entry


@pytest.fixture
def recorder(monkeypatch):
    r = Recorder()
    monkeypatch.setattr(_lib, "lib", lambda: r)
    monkeypatch.setattr(_runtime, "require_gpu", lambda t, what: None)
    for module in (distill, linear, norm):
        monkeypatch.setattr(module, "raw_stream", lambda device: 0)
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


def turned(t):
    """t's values with the first axis innermost."""
    return t.movedim(0, -1).contiguous().movedim(-1, 0)


def lies_at(pointer, pitch, t, ctype=ctypes.c_float):
    """Whether t's rows (2-D) lie at the address, `pitch` elements apart."""
    R, C = t.shape
    flat = np.ctypeslib.as_array((ctype * ((R - 1) * pitch + C)).from_address(pointer))
    rows = np.lib.stride_tricks.as_strided(flat, (R, C), (pitch * flat.itemsize, flat.itemsize))
    return np.array_equal(rows, t.numpy(), equal_nan=ctype is ctypes.c_float)


@pytest.mark.parametrize("lay", [torch.clone, turned])
def test_unpacked_tensors_of_any_layout(recorder, lay):
    # The C entries take rows of unit column stride and contiguous statistics, parts and slopes.
    seen = []
    given = lambda shape: next(t for t in hooks.given if t.shape == shape)

    hooks = Moved(lay)
    s, t, idx = distill_inputs("cpu")
    recorder.look["void_distill_grad"] = lambda a, parts, *_: seen.append(
        lies_at(a.logits, a.ld, s.detach()) and lies_at(a.teacher, a.ldt, t)
        and lies_at(a.index, a.ldi, idx, ctypes.c_int64) and lies_at(parts, 2, given((6, 1, 2))[:, 0]))
    s.requires_grad_()
    with hooks():
        loss = void_amd.distillation_loss(s, t, idx)
    torch.autograd.grad(loss, s)
    assert seen == [True]

    seen.clear()
    hooks = Moved(lay)
    x = torch.randn(6, 40, requires_grad=True)
    recorder.look["void_layer_norm_grad"] = lambda dy, lddy, x_, ldx, w, code, stats, *_: seen.append(
        lies_at(x_, ldx, x.detach()) and lies_at(stats, 2, given((6, 2))))
    with hooks():
        y = void_amd.layer_norm(x)
    torch.autograd.grad(y, x, torch.ones(6, 40))
    assert seen == [True]

    seen.clear()
    hooks = Moved(lay)
    w = torch.randn(16, 40, requires_grad=True)
    recorder.look["void_linear_grad_z"] = lambda dy, lddy, slope, *_: seen.append(lies_at(slope, 16, given((6, 16))))
    recorder.look["void_linear_grad_x"] = lambda dz, ldz, w_, ldw, *_: seen.append(lies_at(w_, ldw, w.detach()))
    recorder.look["void_linear_grad_w"] = lambda dz, ldz, x_, ldx, *_: seen.append(lies_at(x_, ldx, x.detach()))
    with hooks():
        y = void_amd.fused_linear(x, w, None, "silu")
    torch.autograd.grad(y, (x, w), torch.ones(6, 16))
    assert seen == [True] * 3


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


@gpu_only
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K,N", [(5, 40, 24), (70, 130, 33), (150, 203, 117)])
def test_all_three_under_hooks_and_checkpoints(gpu, dtype, M, K, N):
    g = torch.Generator().manual_seed(M)
    leaves = [torch.randn(*shape, generator=g).to(gpu, dtype) for shape in ((M, K), (K,), (K,), (N, K), (N,), (M, N))]
    _, t, idx = distill_inputs(gpu, M, N, 7, dtype)

    def loss(x, nw, nb, w, b, r):
        h = void_amd.layer_norm(x * 1.5, nw, nb)
        y = void_amd.fused_linear(h, w * 0.1, b, "gelu", r * 1.0)
        return void_amd.distillation_loss(y, t * 1.0, idx + 0, 2.0)

    def gradients(around):
        args = [p.detach().requires_grad_() for p in leaves]
        out = around(*args)
        overwritten(gpu)
        out.backward()
        return [p.grad for p in args]

    want = gradients(loss)
    assert all(torch.isfinite(p).all() and p.any() for p in want)

    def hooked(ctx):
        def run(*args):
            with ctx():
                return loss(*args)
        return run
    for around in (hooked(Moved()), hooked(Moved(turned)), hooked(torch.autograd.graph.save_on_cpu),
                   lambda *args: checkpoint(loss, *args, use_reentrant=False)):
        for got, p in zip(gradients(around), want):
            assert torch.equal(got, p)
