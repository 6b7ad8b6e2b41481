"""distillation_loss and distillation_loss_and_grad against a 64-bit
implementation: vocabularies at every kernel variant's edge, few rows and many,
entries that do not count, equal indices, masked and non-finite logits, and the
gradients against the formula's and against differences.

Tolerances: with A = (m - s) / T, an exponential's argument is rounded three
times and its 32-bit sums 64 times, so q is off by 2^-22 (A + log z + 64)
relative and p by 2^-22 (|log p| + 64); a 16-bit gradient is rounded once.
"""

import pytest
import torch

import void_amd

gpu_only = pytest.mark.gpu
E22 = 2.0 ** -22
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def reference(s, t, idx, T):
    """Row losses, the gradient of their sum, whether each row counts, and bounds of the first two."""
    s, t = s.double() / T, t.double() / T
    V = s.shape[1]
    use = (idx >= 0) & (t != float("-inf"))
    some = use.any(1)
    t = torch.where(use, t, float("-inf"))
    top = torch.where(some, t.amax(1), 0.0)[:, None] if t.shape[1] else t.new_zeros(t.shape[0], 1)
    e = torch.exp(t - top)
    total = e.sum(1, keepdim=True)
    p = torch.where(use, e / total, 0.0)
    lp = torch.where(use, t - top - torch.log(total), 0.0)
    m = s.amax(1, keepdim=True)
    z = torch.exp(s - m).sum(1, keepdim=True)
    lz = torch.log(z)
    q = torch.exp(s - m) / z
    at = idx.clamp(min=0).long()
    a = (m - s).gather(1, at)
    live = use & (p > 0)
    loss = T * T * torch.where(live, p * (lp + lz + a), 0.0).sum(1)
    eloss = T * T * torch.where(live, p * (lp.abs() + a + lz + 1), 0.0).sum(1) * 128 * 2.0 ** -24
    P = torch.zeros_like(q).scatter_add_(1, at, p)
    eP = torch.zeros_like(q).scatter_add_(1, at, p * (lp.abs() + 64)) * E22
    eq = q * ((m - s).clamp(max=1e4) + lz + 64) * E22
    keep = some[:, None]
    return (loss, torch.where(keep, T * (q - P), 0.0), some, torch.where(some, eloss, 0.0),
            torch.where(keep, T * (eq + eP), 0.0))


def inputs(gpu, R, V, k, dtype=torch.float32, tdtype=None, seed=0, ragged=False, index=torch.int64):
    g = torch.Generator(device=gpu)
    g.manual_seed(seed)
    s = torch.randn(R, V, generator=g, device=gpu) * 2
    idx = torch.rand(R, V, generator=g, device=gpu).argsort(1)[:, :k]
    t = torch.randn(R, k, generator=g, device=gpu) * 2 + 5
    s = s.scatter_add(1, idx, 0.5 * t)
    if ragged:
        length = torch.randint(0, k + 1, (R, 1), generator=g, device=gpu)
        idx = torch.where(torch.arange(k, device=gpu) < length, idx, -1)
        # In any order, and by a logit of -inf as well.
        order = torch.rand(R, k, generator=g, device=gpu).argsort(1)
        idx, t = idx.gather(1, order), t.gather(1, order)
        t = torch.where((idx < 0) & (torch.arange(k, device=gpu) % 2 == 0), float("-inf"), t)
        idx = torch.where(t == float("-inf"), idx.clamp(min=0), idx)
    return s.to(dtype), t.to(tdtype or dtype), idx.to(index)


def near(got, want, bound, what):
    over = (got.double() - want).abs() - bound - (2.0 ** -24 if got.dtype == torch.float16 else 1e-30)
    assert not torch.isnan(over).any() and over.max() <= 0, f"{what}: {over.max():.3g} over"


def check(s, t, idx, T, scale=1.0):
    loss, grad, some, eloss, egrad = reference(s, t, idx, T)
    n = max(1, int(some.sum()))
    rows = void_amd.distillation_loss(s, t, idx, temperature=T, reduction="none")
    assert rows.dtype == torch.float32
    near(rows, loss, eloss, "row losses")
    sums = 64 * 2.0 ** -24 * loss.abs().sum()
    leaf = s.detach().requires_grad_()
    for reduction, by in (("sum", 1), ("mean", n)):
        out = void_amd.distillation_loss(leaf, t, idx, temperature=T, reduction=reduction)
        near(out.detach(), loss.sum() / by, (eloss.sum() + sums) / by, reduction)
        ds, = torch.autograd.grad(out, leaf, torch.tensor(scale, device=s.device))
        want, bound = grad * scale / by, egrad * scale / by + U[s.dtype] * (grad.abs() + egrad) * scale / by
        assert ds.dtype == s.dtype
        near(ds, want, bound + 2.0 ** -23 * want.abs(), f"gradient of the {reduction}")
        l2, d2 = void_amd.distillation_loss_and_grad(s, t, idx, temperature=T, reduction=reduction, grad_scale=scale)
        near(l2, loss.sum() / by, (eloss.sum() + sums) / by, reduction + " in one call")
        near(d2, want, bound + 2.0 ** -22 * want.abs(), f"gradient of the {reduction} in one call")
    # A gradient per row.
    w = torch.rand(s.shape[0], device=s.device)
    out = void_amd.distillation_loss(leaf, t, idx, temperature=T, reduction="none")
    ds, = torch.autograd.grad(out, leaf, w)
    want = grad * w.double()[:, None]
    near(ds, want, egrad + U[s.dtype] * (want.abs() + egrad) + 2.0 ** -23 * want.abs(), "gradient of rows")


@gpu_only
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,k", [(1, 1, 1), (3, 2, 1), (5, 7, 7), (700, 130, 3), (4, 512, 64), (3, 1024, 9),
                                   (600, 1025, 5), (9, 2049, 65), (2, 5000, 200), (7, 8192, 256), (513, 8200, 20),
                                   (3, 16385, 17), (520, 20001, 33), (1, 33000, 100), (514, 32769, 8), (2, 70001, 64),
                                   (512, 65537, 4)])
def test_against_64_bits(gpu, dtype, R, V, k):
    check(*inputs(gpu, R, V, k, dtype, seed=V), 2.0)


@gpu_only
@pytest.mark.parametrize("dtype,R,V", [(torch.bfloat16, 512, 131073), (torch.float32, 513, 66001), (torch.float16, 1, 300001)])
def test_rows_that_no_register_variant_holds(gpu, dtype, R, V):
    s, t, idx = inputs(gpu, 4, V, 30, dtype)
    pick = torch.arange(R, device=gpu) % 4  # the oracle runs on 4 rows; the rest repeat them
    loss, grad, some, eloss, egrad = reference(s, t, idx, 1.0)
    l2, d2 = void_amd.distillation_loss_and_grad(s[pick], t[pick], idx[pick], reduction="sum")
    near(l2, loss[pick].sum(), 2 * eloss[pick].sum(), "loss")
    near(d2[:4 if R > 3 else R], grad[:4 if R > 3 else R],
         (egrad + (U[dtype] + 2.0 ** -22) * grad.abs())[:4 if R > 3 else R] + U[dtype] * egrad[:4 if R > 3 else R], "gradient")
    for r in range(4, R, 101):
        assert torch.equal(d2[r], d2[r % 4])


@gpu_only
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,k", [(40, 300, 12), (700, 2100, 70), (5, 9000, 130), (3, 40000, 300)])
@pytest.mark.parametrize("T", [0.5, 1.0, 4.0])
def test_lists_of_different_lengths(gpu, dtype, R, V, k, T):
    check(*inputs(gpu, R, V, k, dtype, torch.float32, seed=k, ragged=True, index=torch.int32), T)


@gpu_only
@pytest.mark.parametrize("R,V", [(6, 200), (600, 3000), (4, 20000)])
def test_rows_without_entries(gpu, R, V):
    s, t, idx = inputs(gpu, R, V, 8, torch.bfloat16)
    idx[1::2] = -1
    t[::4] = float("-inf")
    s[1::2, 5] = float("nan")  # not looked at
    s[0, :] = float("inf")
    rows = void_amd.distillation_loss(s, t, idx, reduction="none")
    dead = torch.ones(R, dtype=torch.bool, device=gpu)
    dead[2::4] = False
    assert not rows[dead].any() and (rows[~dead] > 0).all()
    loss, grad = void_amd.distillation_loss_and_grad(s, t, idx)
    leaf = s.detach().requires_grad_()
    out = void_amd.distillation_loss(leaf, t, idx)
    ds, = torch.autograd.grad(out, leaf)
    for g in (grad, ds):
        assert not g[dead].any() and torch.isfinite(g).all() and g[~dead].any(1).all()
    mean = rows.double().sum() / int((~dead).sum())
    assert abs(loss - mean) <= 1e-5 * mean and abs(out.detach() - mean) <= 1e-5 * mean
    idx[:] = -1
    loss, grad = void_amd.distillation_loss_and_grad(s, t, idx)
    assert loss == 0 and not grad.any()
    assert void_amd.distillation_loss(s, t, idx) == 0


@gpu_only
@pytest.mark.parametrize("R,V", [(9, 100), (600, 3000), (3, 20000)])
def test_equal_indices_count_each(gpu, R, V):
    s, t, idx = inputs(gpu, R, V, 40)
    idx[:, 10:20] = idx[:, :10]
    idx[:, 30] = idx[:, 3]
    check(s, t, idx, 1.5)
    a = void_amd.distillation_loss_and_grad(s, t, idx)
    b = void_amd.distillation_loss_and_grad(s, t, idx)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@gpu_only
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V", [(5, 150), (600, 2100), (2, 30000)])
@pytest.mark.parametrize("mask", ["lowest", "-inf"])
def test_masked_logits(gpu, dtype, R, V, mask):
    s, t, idx = inputs(gpu, R, V, 6, dtype)
    low = torch.finfo(dtype).min if mask == "lowest" else float("-inf")
    hide = torch.ones(R, V, dtype=torch.bool, device=gpu)
    hide.scatter_(1, idx, False)
    hide[:, ::3] = False
    hide[:, 1] = True  # a masked place that the teacher knows
    s = s.masked_fill(hide & ~torch.zeros_like(hide).scatter_(1, idx, True), low)
    if R > 4:
        t[3] = torch.finfo(dtype).min  # every entry at the lowest value: all alike
    check(s, t, idx, 0.5)
    # A teacher's entry on a logit of -inf: an infinite loss, a finite gradient.
    s[0, idx[0, 0]] = float("-inf")
    rows = void_amd.distillation_loss(s, t, idx, reduction="none")
    assert rows[0] == float("inf") and torch.isfinite(rows[1:]).all()
    grad = void_amd.distillation_loss_and_grad(s, t, idx, reduction="sum")[1]
    assert torch.isfinite(grad).all() and grad[0, idx[0, 0]] < 0
    s[1] = low  # nothing but masks
    rows = void_amd.distillation_loss(s, t, idx, reduction="none")
    assert torch.isfinite(rows[1]) if mask == "lowest" else torch.isnan(rows[1]) or rows[1] == float("inf")


@gpu_only
@pytest.mark.parametrize("R,V", [(5, 150), (600, 2100), (2, 30000)])
def test_bad_values_stay_in_their_rows(gpu, R, V):
    s, t, idx = inputs(gpu, R, V, 6)
    clean = void_amd.distillation_loss_and_grad(s, t, idx, reduction="sum")[1]
    rows = void_amd.distillation_loss(s, t, idx, reduction="none")
    s2, idx2 = s.clone(), idx.clone()
    s2[0, V // 2] = float("nan")
    idx2[1, 3] = V  # past the vocabulary
    out = void_amd.distillation_loss(s2, t, idx2, reduction="none")
    grad = void_amd.distillation_loss_and_grad(s2, t, idx2, reduction="sum")[1]
    leaf = s2.detach().requires_grad_()
    ds, = torch.autograd.grad(void_amd.distillation_loss(leaf, t, idx2, reduction="sum"), leaf)
    assert out[:2].isnan().all() and torch.equal(out[2:], rows[2:])
    for g in (grad, ds):
        assert g[:2].isnan().all() and torch.isfinite(g[2:]).all()
    assert torch.equal(grad[2:], clean[2:])


@gpu_only
def test_layouts_and_shapes(gpu):
    s, t, idx = inputs(gpu, 12, 1000, 20, torch.bfloat16)
    want = void_amd.distillation_loss_and_grad(s, t, idx)
    place = torch.full((12, 1101), float("nan"), dtype=torch.bfloat16, device=gpu)
    place[:, 1:1001] = s
    wide = place[:, 1:1001]
    got = void_amd.distillation_loss_and_grad(wide, t, idx)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    tt = torch.stack((t, t), 2)[:, :, 0]
    ii = torch.cat((idx, idx), 1)[:, :20]
    for args in ((s.view(3, 4, 1000), t.view(3, 4, 20), idx.view(3, 4, 20)), (s.t().contiguous().t(), tt, ii)):
        got = void_amd.distillation_loss_and_grad(*args)
        assert got[1].shape == args[0].shape
        assert torch.equal(got[0], want[0]) and torch.equal(got[1].reshape(12, 1000), want[1])
    assert void_amd.distillation_loss(s.view(3, 4, 1000), t.view(3, 4, 20), idx.view(3, 4, 20),
                                      reduction="none").shape == (3, 4)
    one = void_amd.distillation_loss(s[0], t[0], idx[0], reduction="none")
    assert one.shape == () and torch.equal(one, void_amd.distillation_loss(s, t, idx, reduction="none")[0])
    for R, V, k in ((0, 50, 3), (4, 50, 0), (0, 0, 0)):
        leaf = torch.randn(R, V, device=gpu, requires_grad=True)
        a = (torch.zeros(R, k, device=gpu), torch.zeros(R, k, dtype=torch.int64, device=gpu))
        out = void_amd.distillation_loss(leaf, *a)
        assert out == 0 and not torch.autograd.grad(out, leaf)[0].any()
        loss, grad = void_amd.distillation_loss_and_grad(leaf, *a)
        assert loss == 0 and grad.shape == (R, V) and not grad.any()


@gpu_only
@pytest.mark.parametrize("R,V", [(4, 300), (2, 9000)])
def test_gradient_against_differences(gpu, R, V):
    s, t, idx = inputs(gpu, R, V, 10)
    leaf = s.detach().requires_grad_()
    grad, = torch.autograd.grad(void_amd.distillation_loss(leaf, t, idx, temperature=2.0, reduction="sum"), leaf)
    d = torch.randn_like(s)
    h = 2.0 ** -4
    f = lambda x: void_amd.distillation_loss(x, t, idx, temperature=2.0, reduction="none").double().sum()
    slope = (f(s + h * d) - f(s - h * d)) / (2 * h)
    want = (grad.double() * d.double()).sum()
    # Third derivatives are below |d|^3 / T, losses 2^-18 of their size apart.
    top = d.abs().max()
    assert (slope - want).abs() <= R * (h * h / 6 * top ** 3 / 2 + 2.0 ** -18 * 20 / h)


@gpu_only
def test_streams_and_graphs(gpu):
    s, t, idx = inputs(gpu, 300, 9000, 16, torch.bfloat16)
    want = void_amd.distillation_loss_and_grad(s, t, idx)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = void_amd.distillation_loss_and_grad(s, t, idx)
    st.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = void_amd.distillation_loss_and_grad(s, t, idx)
    for _ in range(3):
        got[1].zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(void_amd.distillation_loss_and_grad(s, t, idx)[1], want[1])


@gpu_only
@pytest.mark.parametrize("R,V", [(1, 9000), (15, 20001), (16, 40000), (17, 40000), (40, 9000)])
def test_few_rows_give_the_same_sum_each_time(gpu, R, V):
    s, t, idx = inputs(gpu, R, V, 33, torch.bfloat16, seed=R, ragged=True)
    idx[0] = -1  # a row that does not count arrives too
    check(s, t, idx, 2.0)
    want = void_amd.distillation_loss_and_grad(s, t, idx)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = void_amd.distillation_loss_and_grad(s, t, idx)
    for _ in range(5):
        got[0].fill_(7.0), got[1].zero_()
        g.replay()
        torch.cuda.synchronize()
        again = void_amd.distillation_loss_and_grad(s, t, idx)
        for out in (got, again):
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@gpu_only
def test_forward_mode_and_second_derivatives_are_refused(gpu):
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.randn(4, 16, device=gpu), torch.ones(4, 16, device=gpu))
        with pytest.raises((RuntimeError, NotImplementedError)):
            void_amd.distillation_loss(x, torch.zeros(4, 2, device=gpu), torch.zeros(4, 2, dtype=torch.int64, device=gpu))
    x = torch.randn(4, 16, device=gpu, requires_grad=True)
    g, = torch.autograd.grad(void_amd.distillation_loss(x, torch.zeros(4, 2, device=gpu), torch.zeros(4, 2, dtype=torch.int64, device=gpu)).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@gpu_only
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,V", [(5, 7), (600, 513), (600, 2051), (520, 9001), (513, 33001), (3, 20003), (18, 20003)])
@pytest.mark.parametrize("shift,gap", [(1, 1), (1, 2), (2, 3)])
def test_rows_between_dwords(gpu, dtype, R, V, shift, gap):
    # What lies beside the rows is never seen.
    s, t, idx = inputs(gpu, R, V, 5, dtype, seed=V, ragged=True)
    buf = torch.full((R * (V + gap) + 8,), float("inf"), device=gpu, dtype=dtype)
    rows = buf[shift:shift + R * (V + gap)].view(R, V + gap)[:, :V].copy_(s)
    check(rows, t, idx, 2.0)


@gpu_only
def test_offsets_past_31_bits(gpu):
    V, k = 131072, 20
    R = (1 << 31) // V + 3
    s, t, idx = inputs(gpu, 16, V, k, torch.bfloat16)
    s, t, idx = (a.repeat(-(-R // 16), 1)[:R].contiguous() for a in (s, t, idx))
    ends = s[-20:], t[-20:], idx[-20:]
    want, grad, _, bound, egrad = reference(*ends, 2.0)
    near(void_amd.distillation_loss(s, t, idx, temperature=2.0, reduction="none")[-20:], want, bound, "row losses")
    by = egrad + U[s.dtype] * (grad.abs() + egrad) + 2.0 ** -22 * grad.abs()
    near(void_amd.distillation_loss_and_grad(s, t, idx, 2.0, "sum")[1][-20:], grad, by, "gradient in one call")
    s.requires_grad_()
    ds, = torch.autograd.grad(void_amd.distillation_loss(s, t, idx, 2.0, "sum"), s)
    near(ds[-20:], grad, by, "gradient")


def test_refusals():
    s, t, i = torch.randn(2, 50), torch.randn(2, 4), torch.zeros(2, 4, dtype=torch.int64)
    for call in (void_amd.distillation_loss, void_amd.distillation_loss_and_grad):
        with pytest.raises(RuntimeError, match="GPU"):
            call(s, t, i)
        with pytest.raises(TypeError):
            call(s.double(), t, i)
        with pytest.raises(TypeError):
            call(s, t, i.to(torch.int16))
        with pytest.raises(TypeError):
            call(s, t.to(torch.int32), i)
        for bad in ((s, t[:, :3], i), (s, t[:1], i[:1]), (s[0], t, i), (s, t[0, 0], i[0, 0])):
            with pytest.raises(ValueError):
                call(*bad)
        for V in (1 << 30, (1 << 32) + 4):  # columns that 31 or 32 bits do not hold
            with pytest.raises(ValueError, match="long"):
                call(torch.zeros(1).expand(2, V), t, i)
        with pytest.raises(ValueError, match="1024"):
            call(s, torch.zeros(2, 1025), torch.zeros(2, 1025, dtype=torch.int64))
        for T in (0.0, -1.0, float("nan"), float("inf")):
            with pytest.raises(ValueError, match="temperature"):
                call(s, t, i, temperature=T)
        with pytest.raises(ValueError, match="reduction"):
            call(s, t, i, reduction="batchmean")
    with pytest.raises(ValueError, match="reduction"):
        void_amd.distillation_loss_and_grad(s, t, i, reduction="none")


def test_abi_refusals():
    import ctypes
    from void_amd import _lib
    lib = _lib.lib()
    at = 1 << 20  # a non-null, aligned address that is never read: every call below is refused
    base = dict(logits=at, ld=50, teacher=at, ldt=4, index=at, ldi=4, rows=2, vocab=50, k=4, dtype=0, teacher_dtype=0,
                index_bytes=8, temperature=1.0)
    for bad, code in ((dict(rows=-1), -1), (dict(k=1025), -2), (dict(vocab=1 << 30, ld=1 << 30), -2), (dict(dtype=3), -2), (dict(index_bytes=2), -2),
                      (dict(temperature=0.0), -1), (dict(logits=None), -1), (dict(index=at + 4), -1), (dict(ld=-1), -1)):
        a = _lib.DistillArgs(**{**base, **bad})
        assert lib.void_distill_loss(ctypes.byref(a), at, at, at, None) == code, bad
    a = _lib.DistillArgs(**base)
    assert lib.void_distill_step(ctypes.byref(a), 1, 1.0, at, at, 50, None, 0, None) == -4
    assert lib.void_distill_step(ctypes.byref(a), 1, 1.0, at, at, 49, at, 1 << 20, None) == -1
    assert lib.void_distill_slices(8, 131072) == 32 and lib.void_distill_slices(4096, 131072) == 1
