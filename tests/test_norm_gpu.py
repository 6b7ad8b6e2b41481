"""layer_norm against a 64-bit implementation: widths at every kernel variant's
edge, pitches and unaligned rows, parameter types, rows with infinities and
NaN, streams, and its gradients against the formula's and against differences.

Tolerances: a stored 16-bit value is rounded once (U relative); a row's 32-bit
sums add at most 16 values a thread and then a tree, 64 roundings in all with
the arithmetic around them; a column's sum adds one rounding a row.
"""

import pytest
import torch

import void_amd

gpu_only = pytest.mark.gpu
EPS32 = 2.0 ** -24
U = {torch.float32: EPS32, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def reference(x, w, b, dy, eps=1e-5):
    """y, dx, dw, db and a bound for each from 64-bit values."""
    dt = x.dtype
    x, dy = x.double(), dy.double()
    w = torch.ones(x.shape[1], device=x.device).double() if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    mu = x.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((x - mu) ** 2).mean(1, keepdim=True) + eps)
    h = (x - mu) * r
    g = dy * w
    y = h * w + b
    c1, c2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    dx, dw, db = r * (g - c1 - h * c2), (dy * h).sum(0), dy.sum(0)
    # What an error of 64 roundings in the sums does to h, and from there on.
    off = r * x.abs().mean(1, keepdim=True) + r * x.abs()
    eh = 64 * EPS32 * (h.abs() + off)
    ey = eh * w.abs() + 4 * EPS32 * (y.abs() + b.abs()) + U[dt] * y.abs()
    mg = g.abs().mean(1, keepdim=True)
    mh = (g.abs() * (h.abs() + off)).mean(1, keepdim=True)
    edx = 128 * EPS32 * r * (g.abs() + mg + (h.abs() + off + 1) * (mh + mg)) + U[dt] * dx.abs()
    rows = x.shape[0]
    edw = (128 + rows) * EPS32 * (dy.abs() * (h.abs() + off)).sum(0)
    edb = (128 + rows) * EPS32 * dy.abs().sum(0)
    return (y, dx, dw, db), (ey, edx, edw, edb)


def close(got, want, bound, what):
    tiny = 2.0 ** -24 if got.dtype == torch.float16 else 1e-37  # fp16 below its normal numbers
    over = (got.double() - want).abs() - bound - tiny
    assert got.shape == want.shape and not torch.isnan(over).any() and over.max() <= 0, f"{what}: {over.max():.3g} over"


def check(x, w, b, dy):
    x, dy = x.detach().requires_grad_(), dy.detach()
    params = [p.detach().requires_grad_() for p in (w, b) if p is not None]
    it = iter(params)
    y = void_amd.layer_norm(x, next(it) if w is not None else None, next(it) if b is not None else None)
    assert y.dtype == x.dtype and y.shape == x.shape
    grads = torch.autograd.grad(y, [x, *params], dy)
    (ry, rx, rw, rb), (ey, ex, ew, eb) = reference(x.detach(), w, b, dy)
    close(y.detach(), ry, ey, "y")
    close(grads[0], rx, ex, "dx")
    it = iter(grads[1:])
    if w is not None:
        dw = next(it)
        assert dw.dtype == w.dtype
        close(dw, rw, ew + U[w.dtype] * rw.abs(), "dw")
    if b is not None:
        close(next(it), rb, eb + U[b.dtype] * rb.abs(), "db")


def inputs(gpu, dtype, R, C, seed=0, pdtype=None):
    g = torch.Generator(device=gpu)
    g.manual_seed(seed)
    x = (torch.randn(R, C, generator=g, device=gpu) * 2 + 0.5).to(dtype)
    w = (1 + 0.2 * torch.randn(C, generator=g, device=gpu)).to(pdtype or dtype)
    b = (0.2 * torch.randn(C, generator=g, device=gpu)).to(pdtype or dtype)
    return x, w, b, torch.randn(R, C, generator=g, device=gpu).to(dtype)


@gpu_only
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,C", [(1, 1), (3, 1), (1, 7), (5, 8), (37, 63), (130, 64), (33, 65), (65, 129), (9, 255),
                                 (70, 512), (31, 513), (5, 1024), (600, 1025), (7, 2047), (3, 2049), (520, 4096),
                                 (4, 5001), (2, 8192), (5, 8193), (300, 9001), (3, 16384), (5, 16385), (2, 40001)])
def test_against_64_bits(gpu, dtype, R, C):
    check(*inputs(gpu, dtype, R, C, R + C))


@gpu_only
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,C", [(9, 200), (17, 1500), (3, 4097), (2, 20000)])
def test_fp32_parameters(gpu, dtype, R, C):
    check(*inputs(gpu, dtype, R, C, 1, torch.float32))


@gpu_only
@pytest.mark.parametrize("have", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("C", [96, 3000, 17000])
def test_optional_parameters(gpu, have, C):
    x, w, b, dy = inputs(gpu, torch.bfloat16, 6, C)
    check(x, w if have[0] else None, b if have[1] else None, dy)


@gpu_only
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C,pitch,shift", [(130, 131, 1), (1000, 1009, 3), (2500, 2501, 1), (6000, 6007, 5)])
def test_pitch_and_alignment(gpu, dtype, C, pitch, shift):
    x, w, b, dy = inputs(gpu, dtype, 11, C)
    # Whatever lies between the rows is not read.
    place = torch.full((11 * pitch + shift,), float("nan"), dtype=dtype, device=gpu)
    xs = place[shift:].view(11, pitch)[:, :C]
    xs.copy_(x)
    gs = place.clone()[shift:].view(11, pitch)[:, :C]
    gs.copy_(dy)
    assert torch.equal(void_amd.layer_norm(xs, w, b), void_amd.layer_norm(x, w, b))
    a = xs.detach().requires_grad_()
    c = x.detach().requires_grad_()
    da, = torch.autograd.grad(void_amd.layer_norm(a, w, b), a, gs)
    dc, = torch.autograd.grad(void_amd.layer_norm(c, w, b), c, dy)
    assert torch.equal(da, dc)


@gpu_only
def test_shapes_and_broadcast_inputs(gpu):
    x, w, b, _ = inputs(gpu, torch.float32, 24, 40)
    y = void_amd.layer_norm(x, w, b)
    assert torch.equal(void_amd.layer_norm(x.view(2, 3, 4, 40), w, b), y.view(2, 3, 4, 40))
    assert torch.equal(void_amd.layer_norm(x[3], w, b), y[3])
    assert torch.equal(void_amd.layer_norm(x.t().contiguous().t(), w, b), y)
    # One row repeated: each gradient of it counts.
    row = x[:1].detach().requires_grad_()
    out = void_amd.layer_norm(row.expand(24, 40), w, b)
    assert torch.equal(out, y[:1].expand(24, 40))
    out.sum().backward()  # a gradient of stride 0
    check_row = x[:1].double().requires_grad_()
    torch.nn.functional.layer_norm(check_row, (40,), w.double(), b.double()).sum().mul(24).backward()
    assert (row.grad - check_row.grad).abs().max() <= 24 * 512 * EPS32


@gpu_only
@pytest.mark.parametrize("shape", [(0, 16), (3, 0), (0, 0), (0, 20000)])
def test_empty(gpu, shape):
    x = torch.empty(shape, device=gpu, requires_grad=True)
    w, b = (torch.ones(shape[1], device=gpu, requires_grad=True) for _ in range(2))
    y = void_amd.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert y.shape == dx.shape == shape and not dw.any() and not db.any() and dw.shape == (shape[1],)


@gpu_only
@pytest.mark.parametrize("shape", [(2, 3, 0), (0, 3, 5), (2, 0, 5), (2, 0, 0)])
def test_empty_axes_of_more_dimensions(gpu, shape):
    x = torch.empty(shape, device=gpu, requires_grad=True)
    w, b = (torch.ones(shape[-1], device=gpu, requires_grad=True) for _ in range(2))
    y = void_amd.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert y.shape == dx.shape == shape and not dw.any() and not db.any() and dw.shape == db.shape == (shape[-1],)


def test_rows_of_empty_tensors():
    from void_amd import _runtime
    for shape, rows in (((2, 3, 0), (6, 0)), ((0, 3, 5), (0, 5)), ((2, 0, 0), (0, 0)), ((0,), (1, 0)), ((5,), (1, 5))):
        assert _runtime.flat_rows(torch.empty(shape)).shape == rows


@gpu_only
@pytest.mark.parametrize("C", [50, 3000, 17000])
def test_non_finite_rows_stay_alone(gpu, C):
    x, w, b, dy = inputs(gpu, torch.float32, 8, C)
    clean = void_amd.layer_norm(x, w, b)
    x[2, C // 2], x[5, C - 1] = float("nan"), float("inf")
    y = void_amd.layer_norm(x, w, b)
    assert y[2].isnan().all() and y[5].isnan().all()
    keep = [0, 1, 3, 4, 6, 7]
    assert torch.equal(y[keep], clean[keep])


@gpu_only
def test_offset_costs_no_precision(gpu):
    x, w, b, dy = inputs(gpu, torch.float32, 16, 3000)
    check(x + 1000.0, w, b, dy)
    check(torch.full_like(x, 3.0), w, b, dy)  # no variance at all


@gpu_only
def test_gradients_against_differences(gpu):
    x, w, b, dy = inputs(gpu, torch.float32, 5, 70)
    f = lambda *a: (void_amd.layer_norm(*a).double() * dy.double()).sum()
    args = [t.detach().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(void_amd.layer_norm(*args), args, dy)
    for i in range(3):
        d = torch.randn_like(args[i])
        h = 2.0 ** -6
        up, down = [a.detach() for a in args], [a.detach() for a in args]
        up[i], down[i] = args[i].detach() + h * d, args[i].detach() - h * d
        slope = (f(*up) - f(*down)) / (2 * h)
        want = (grads[i].double() * d.double()).sum()
        # Truncation h^2, and 32-bit results 2^-24 apart over 2 h.
        scale = (dy.abs() * d.abs().max()).sum()
        assert (slope - want).abs() <= scale * (h * h + 16 * EPS32 / h)


@gpu_only
def test_stream_repeat_and_partial_gradients(gpu):
    x, w, b, dy = inputs(gpu, torch.bfloat16, 700, 1000)
    a = [t.detach().requires_grad_() for t in (x, w, b)]
    first = torch.autograd.grad(void_amd.layer_norm(*a), a, dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = torch.autograd.grad(void_amd.layer_norm(*a), a, dy)
    s.synchronize()
    for p, q in zip(first, again):
        assert torch.equal(p, q)
    for i in range(3):  # one gradient alone has the same bits
        c = [t.detach() for t in (x, w, b)]
        c[i].requires_grad_()
        assert torch.equal(torch.autograd.grad(void_amd.layer_norm(*c), c[i], dy)[0], first[i])
    m = void_amd.LayerNorm(1000, dtype=torch.bfloat16, device=gpu)
    assert torch.equal(m(x), void_amd.layer_norm(x, torch.ones_like(w), torch.zeros_like(b)))


@gpu_only
def test_graph_replays(gpu):
    x, w, b, _ = inputs(gpu, torch.bfloat16, 64, 4096)
    want = void_amd.layer_norm(x, w, b)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = void_amd.layer_norm(x, w, b)
    for _ in range(3):
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        assert torch.equal(void_amd.layer_norm(x, w, b), want)


@gpu_only
def test_forward_mode_and_second_derivatives_are_refused(gpu):
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.randn(4, 16, device=gpu), torch.ones(4, 16, device=gpu))
        with pytest.raises((RuntimeError, NotImplementedError)):
            void_amd.layer_norm(x)
    x = torch.randn(4, 16, device=gpu, requires_grad=True)
    g, = torch.autograd.grad(void_amd.layer_norm(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@gpu_only
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("C", [5, 63, 257, 1500, 4097, 16383, 16391])
@pytest.mark.parametrize("shift,gap", [(0, 1), (1, 0), (1, 1), (3, 2)])
def test_rows_between_dwords(gpu, dtype, C, shift, gap):
    # What lies beside the rows is never seen.
    x, w, b, dy = inputs(gpu, dtype, 6, C, C + shift)

    def spread(t, at):
        pitch = C + gap
        buf = torch.full((6 * pitch + 8,), float("nan"), device=gpu, dtype=dtype)
        return buf[at:at + 6 * pitch].view(6, pitch)[:, :C].copy_(t)
    check(spread(x, shift), w, b, spread(dy, shift))
    check(spread(x, shift), w, b, dy)
    check(x, w, b, spread(dy, 1))


@gpu_only
def test_offsets_past_31_bits(gpu):
    R, C = (1 << 31) // 8192 + 5, 8192
    x = torch.randn(64, C, device=gpu, dtype=torch.bfloat16).repeat(-(-R // 64), 1)[:R]
    w, b = torch.randn(2, C, device=gpu, dtype=torch.bfloat16)
    x.requires_grad_()
    y = void_amd.layer_norm(x, w, b)
    dx, = torch.autograd.grad(y, x, x.detach())
    ends = [t.detach()[-70:] for t in (x, y, dx)]
    (ry, rx, _, _), (ey, ex, _, _) = reference(ends[0], w, b, ends[0])
    close(ends[1], ry, ey, "y")
    close(ends[2], rx, ex, "dx")


@gpu_only
def test_rows_of_more_columns_than_one_grid_axis_sums(gpu):
    # 2^26 groups of 64 columns' sums are more than 2^32 threads along one axis of a grid.
    C = (1 << 27) + 37
    x = torch.randn(C, device=gpu, dtype=torch.bfloat16)[None]
    dy = torch.randn(C, device=gpu, dtype=torch.bfloat16)[None]
    w, b = (torch.randn(C, device=gpu, dtype=torch.bfloat16).requires_grad_() for _ in range(2))
    dw, db = torch.autograd.grad(void_amd.layer_norm(x, w, b), (w, b), dy)
    # One row: its own terms, at both ends and at the places that would be another's.
    mean, var = x.double().mean(), x.double().var(correction=0)
    for part in (slice(0, 70), slice((1 << 26) - 40, (1 << 26) + 40), slice(C - 70, C)):
        h = (x[0, part].double() - mean) / torch.sqrt(var + 1e-5)
        want = dy[0, part].double() * h
        # Sums of 2^27 values in 1024 threads: 2^14 terms each; the row's mean is near 0.
        bound = (1 << 15) * EPS32 * dy[0, part].double().abs() * (h.abs() + 1) + U[torch.bfloat16] * want.abs()
        close(dw[part], want, bound, "dw")
        assert torch.equal(db[part], dy[0, part])


def test_refusals():
    x = torch.randn(2, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        void_amd.layer_norm(x)
    with pytest.raises(TypeError):
        void_amd.layer_norm(x.double())
    with pytest.raises(TypeError):
        void_amd.layer_norm(x, torch.ones(8, dtype=torch.int32))
    with pytest.raises(ValueError):
        void_amd.layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError):
        void_amd.layer_norm(x, None, torch.ones(1))
    with pytest.raises(ValueError):
        void_amd.layer_norm(torch.tensor(1.0))
    for C in (1 << 30, (1 << 32) + 4):  # columns that 31 or 32 bits do not hold
        with pytest.raises(ValueError, match="long"):
            void_amd.layer_norm(torch.zeros(1).expand(C))


def test_abi_refusals():
    from void_amd import _lib
    lib = _lib.lib()
    one = 1 << 20  # a non-null, aligned address that is never read: every call below is refused
    ok = dict(x=one, ldx=8, w=None, b=None, pd=0, rows=2, cols=8, eps=1e-5, dt=0, y=one, ldy=8, stats=None, stream=None)
    for bad, code in ((dict(x=None), -1), (dict(y=None), -1), (dict(rows=-1), -1), (dict(ldy=7), -1), (dict(x=one + 2), -1),
                      (dict(dt=3), -2), (dict(cols=1 << 30, ldx=1 << 30, ldy=1 << 30), -2), (dict(pd=1), -2), (dict(stats=one + 4), -1)):
        assert lib.void_layer_norm(*{**ok, **bad}.values()) == code, bad
    args = [one, 8, one, 8, None, 0, one, 2, 8, 0, one, 8, one, one, None, 0, None]
    assert lib.void_layer_norm_grad(*args) == -4  # no workspace
    assert lib.void_layer_norm_grad_workspace_bytes(2, 8, 0) > 0
