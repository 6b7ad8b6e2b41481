"""fused_linear against a 64-bit implementation: sizes at every tile's and
variant's edge, split sums, unaligned and strided operands, activations,
residuals, non-finite values, and its gradients against the formula's and
against differences.

Tolerances: a sum of K exact products rounds at most K + 32 times in fp32 (in
any order), with 16-bit inputs each stored value rounds once more; an
activation's error is that of its argument, times a slope of at most 1.13, and
2^-20 of its size; dZ is rounded to the inputs' type before the gradients'
products, and a 16-bit layer's slope is kept to 2^-16.
"""

import pytest
import torch

import void_amd

gpu_only = pytest.mark.gpu
EPS32 = 2.0 ** -24
U = {torch.float32: EPS32, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def act(z, name):
    """activation, its slope."""
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "gelu":
        u = 0.7978845608 * (z + 0.044715 * z ** 3)
        t = torch.tanh(u)
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * 0.7978845608 * (1 + 0.134145 * z * z)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def reference(x, w, b, r, dy, name):
    dt = x.dtype
    x, w = x.double(), w.double()
    M, K = x.shape
    z, ez = x @ w.t(), (K + 32) * EPS32 * (x.abs() @ w.abs().t())
    if b is not None:
        z = z + b.double()
        ez = ez + 2 * EPS32 * (z.abs() + b.double().abs())
    y, slope = act(z, name)
    ey = 1.13 * ez + (2.0 ** -20 * z.abs() if name in ("gelu", "silu") else 0)
    if r is not None:
        y = y + r.double()
    ey = ey + 2 * EPS32 * y.abs() + U[dt] * y.abs()
    if dy is None:
        return (y,), (ey,)
    dy = dy.double()
    # |act''| is at most 1.13 (gelu), 0.5 (silu); a relu's slope may flip within ez of 0.
    es = {"none": 0 * ez, "relu": (z.abs() <= ez).double(), "gelu": 1.13 * ez + 2.0 ** -19,
          "silu": 0.5 * ez + 2.0 ** -19}[name]
    if dt != torch.float32 and name != "none":
        es = es + 2.0 ** -16
    dz = dy * slope
    edz = dy.abs() * es + (U[dt] * dz.abs() if name != "none" else 0)
    N = w.shape[0]
    edx = edz @ w.abs() + (N + 32) * EPS32 * (dz.abs() @ w.abs())
    edw = edz.t() @ x.abs() + (M + 32) * EPS32 * (dz.abs().t() @ x.abs())
    dx, dw, db = dz @ w, dz.t() @ x, dz.sum(0)
    edb = (dy.abs() * es).sum(0) + (M + 32) * EPS32 * dz.abs().sum(0)
    return (y, dx, dw, db), (ey, edx + U[dt] * dx.abs(), edw + U[dt] * dw.abs(), edb)


def close(got, want, bound, what):
    over = (got.double() - want).abs() - bound - (2.0 ** -24 if got.dtype == torch.float16 else 1e-30)
    assert got.shape == want.shape and not torch.isnan(over).any() and (not over.numel() or over.max() <= 0), \
        f"{what}: {over.max():.3g} over"


def inputs(gpu, M, N, K, dtype, seed=0):
    g = torch.Generator(device=gpu)
    g.manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device=gpu)
    return (rnd(M, K).to(dtype), (rnd(N, K) / max(K, 1) ** 0.5).to(dtype), rnd(N).to(dtype), rnd(M, N).to(dtype),
            rnd(M, N).to(dtype))


def check(x, w, b, r, dy, name):
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r) if t is not None]
    it = iter(leaves)
    a = [next(it) if t is not None else None for t in (x, w, b, r)]
    y = void_amd.fused_linear(a[0], a[1], a[2], name, a[3])
    plain = void_amd.fused_linear(x, w, b, name, r)
    assert y.dtype == x.dtype and torch.equal(y.detach(), plain)
    want, bound = reference(x, w, b, r, dy, name)
    close(y.detach(), want[0], bound[0], "y")
    grads = dict(zip([n for n, t in zip("xwbr", (x, w, b, r)) if t is not None],
                     torch.autograd.grad(y, leaves, dy)))
    close(grads["x"], want[1], bound[1], "dx")
    close(grads["w"], want[2], bound[2], "dw")
    if b is not None:
        assert grads["b"].dtype == b.dtype
        close(grads["b"], want[3], bound[3] + U[b.dtype] * want[3].abs(), "db")
    if r is not None:
        assert torch.equal(grads["r"], dy)


SIZES = [(1, 1, 1), (1, 17, 40), (3, 5, 7), (16, 16, 32), (17, 33, 129), (40, 100, 300), (64, 64, 64), (65, 8, 8),
         (70, 130, 72), (128, 128, 64), (129, 127, 65), (200, 300, 500), (256, 256, 256), (300, 520, 1030),
         (513, 257, 264), (100, 40, 5000), (1000, 24, 40)]


@gpu_only
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_against_64_bits(gpu, dtype, M, N, K):
    x, w, b, r, dy = inputs(gpu, M, N, K, dtype, M + N + K)
    check(x, w, b, r, dy, "gelu")
    check(x, w, b, None, dy, "none")


@gpu_only
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("M,N,K", [(9, 50, 70), (150, 140, 136)])
def test_epilogues(gpu, dtype, name, M, N, K):
    x, w, b, r, dy = inputs(gpu, M, N, K, dtype)
    for bb, rr in ((None, None), (b, None), (None, r), (b.float() if dtype != torch.float32 else b.half(), r)):
        if bb is not None and bb.dtype == torch.float16 and dtype == torch.float32:
            # Another 16-bit type is widened, exactly.
            assert torch.equal(void_amd.fused_linear(x, w, bb, name), void_amd.fused_linear(x, w, bb.float(), name))
            continue
        check(x, w, bb, rr, dy, name)


@gpu_only
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(4096, 4096, 512), (2049, 4100, 1000), (300, 4096, 14336), (96, 96, 20000)])
def test_larger_tiles_and_split_sums(gpu, dtype, M, N, K):
    x, w, b, r, _ = inputs(gpu, M, N, K, dtype)
    want, bound = reference(x, w, b, r, None, "silu")
    close(void_amd.fused_linear(x, w, b, "silu", r), want[0], bound[0], "y")


@gpu_only
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(64, 20000, 96), (16, 9000, 1000), (33, 163, 4736), (1, 8192, 11054)])
def test_few_tokens(gpu, dtype, M, N, K):
    x, w, b, r, _ = inputs(gpu, M, N, K, dtype)
    want, bound = reference(x, w, b, r, None, "gelu")
    got = void_amd.fused_linear(x, w, b, "gelu", r)
    close(got, want[0], bound[0], "y")
    # Of any alignment: rows that start anywhere, NaN around them.
    def moved(t):
        place = torch.full((t.shape[0] * (t.shape[1] + 3) + 1,), float("nan"), dtype=dtype, device=gpu)
        view = place[1:].view(t.shape[0], t.shape[1] + 3)[:, :t.shape[1]]
        view.copy_(t)
        return view
    close(void_amd.fused_linear(moved(x), moved(w), b, "gelu", moved(r)), want[0], bound[0], "y of unaligned rows")


@gpu_only
@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(gpu, dtype):
    M, N, K = 150, 203, 117
    x, w, b, r, dy = inputs(gpu, M, N, K, dtype)
    want = void_amd.fused_linear(x, w, b, "relu", r)
    place = lambda t: torch.cat((torch.full_like(t[:, :1], float("nan")), t, torch.full_like(t[:, :4], float("nan"))), 1)[
        :, 1:1 + t.shape[1]]
    turned = lambda t: t.t().contiguous().t()
    for f in (place, turned):
        assert torch.equal(void_amd.fused_linear(f(x), f(w), b, "relu", f(r)), want)
        a = [t.detach().requires_grad_() for t in (f(x), f(w), b, f(r))]
        c = [t.detach().requires_grad_() for t in (x, w, b, r)]
        ga = torch.autograd.grad(void_amd.fused_linear(a[0], a[1], a[2], "relu", a[3]), a, f(dy))
        gc = torch.autograd.grad(void_amd.fused_linear(c[0], c[1], c[2], "relu", c[3]), c, dy)
        for p, q in zip(ga, gc):
            assert torch.equal(p, q)
    y = void_amd.fused_linear(x.view(3, 50, K), w, b, "relu", r.view(3, 50, N))
    assert y.shape == (3, 50, N) and torch.equal(y.view(M, N), want)
    one = void_amd.fused_linear(x[0], w, b, "relu", r[0])
    assert one.shape == (N,)
    # One row repeated, a residual row repeated, and a gradient of stride 0.
    rep = void_amd.fused_linear(x[:1].expand(M, K), w, b, "relu", r[:1].expand(M, N))
    assert torch.equal(rep, rep[:1].expand(M, N))
    few = void_amd.fused_linear(x[:1].expand(5, K), w, b, "relu", r[:1].expand(5, N))
    assert torch.equal(few, few[:1].expand(5, N))
    leaf = x.detach().requires_grad_()
    ds, = torch.autograd.grad(void_amd.fused_linear(leaf, w).sum(), leaf)
    d2, = torch.autograd.grad(void_amd.fused_linear(leaf, w), leaf, torch.ones(M, N, dtype=dtype, device=gpu))
    assert torch.equal(ds, d2)


@gpu_only
@pytest.mark.parametrize("shape", [(0, 5, 8), (3, 0, 8), (3, 5, 0), (200, 5, 0), (0, 0, 0), (200, 0, 16)])
def test_empty(gpu, shape):
    M, N, K = shape
    x, w, b, r, dy = (t.requires_grad_() for t in inputs(gpu, M, N, K, torch.bfloat16))
    y = void_amd.fused_linear(x, w, b, "gelu", r)
    grads = torch.autograd.grad(y, (x, w, b, r), dy.detach())
    assert y.shape == (M, N) and [g.shape for g in grads] == [t.shape for t in (x, w, b, r)]
    if K == 0 and M and N:
        z = torch.nn.functional.gelu(b.detach().double(), approximate="tanh") + r.detach().double()
        close(y.detach(), z, 2.0 ** -8 * z.abs() + 2.0 ** -18, "y")
        assert grads[0].numel() == grads[1].numel() == 0
    if M == 0:
        assert not grads[1].any() and not grads[2].any()
    if N == 0:
        assert not grads[0].any()


@gpu_only
@pytest.mark.parametrize("M", [5, 150])
@pytest.mark.parametrize("name", ["none", "relu", "gelu", "silu"])
def test_non_finite_values_stay_alone(gpu, M, name):
    x, w, b, r, dy = inputs(gpu, M, 100, 64, torch.float16)
    clean = void_amd.fused_linear(x, w, b, name, r)
    x[2, 5], r[4, 7] = float("nan"), float("inf")
    w2, b2 = w.clone(), b.clone()
    b2[9] = float("nan")
    y = void_amd.fused_linear(x, w2, b2, name, r)
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[2], keep[4, 7], keep[:, 9] = False, False, False
    assert torch.equal(y[keep], clean[keep]) and y[2].isnan().all() and y[:, 9].isnan().all()
    assert y[4, 7] == float("inf")
    # Large arguments: the activation's limits, and slopes of 0 and 1.
    big = torch.tensor([[6e4], [-6e4]], dtype=torch.float16, device=gpu).repeat(M, 1).requires_grad_()
    one = torch.ones(1, 1, dtype=torch.float16, device=gpu)
    out = void_amd.fused_linear(big, one, None, name)
    g, = torch.autograd.grad(out, big, torch.ones_like(out))
    low = 0.0 if name != "none" else -6e4
    assert (out[0::2] == 6e4).all() and (out[1::2] == torch.tensor(low, dtype=torch.float16)).all()
    assert (g[0::2] == 1).all() and (g[1::2] == (1 if name == "none" else 0)).all()


@gpu_only
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [7, 130])
@pytest.mark.parametrize("name,low,high", [("silu", -16.0, -7.0), ("gelu", -4.8, -3.2)])
def test_saturated_units_keep_their_gradients(gpu, dtype, M, name, low, high):
    # Units whose slope is 2^-24 to 0.03: relative bounds.  The slope is kept to 2^-10 of
    # itself from 2^-29 on; an error of z changes it by at most 8 of that relative (2 u' + 1 <=
    # 8 for gelu, 1 for silu); its own arithmetic rounds an exponent below 32 in 2^-24 steps a
    # few times, 2^-17 in all; dZ rounds once more before the products.
    N, K = 48, 64
    x, w, _, _, dy = inputs(gpu, M, N, K, dtype, 5)
    w = w * 0.125
    b = torch.linspace(low, high, N, device=gpu).to(dtype)
    dy = dy.sign() * (dy.abs() + 0.25) * 8192  # as a loss scaler: dZ stays a normal fp16 value
    a = [t.detach().requires_grad_() for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(void_amd.fused_linear(*a, name), a, dy)
    X, W, D = x.double(), w.double(), dy.double()
    z = X @ W.t() + b.double()
    ez = (K + 32) * EPS32 * (X.abs() @ W.abs().t()) + 2 * EPS32 * (z.abs() + b.double().abs())
    if name == "silu":
        s = torch.sigmoid(z)
        slope = s * (1 + z * torch.sigmoid(-z))
    else:
        v = 1.5957691216 * (z + 0.044715 * z ** 3)
        s = torch.sigmoid(v)
        slope = s * (1 + z * torch.sigmoid(-v) * 1.5957691216 * (1 + 0.134145 * z * z))
    assert (slope < 0).all() and slope.abs().min() > 2.0 ** -24 and slope.abs().max() < 0.03
    dz = D * slope
    es = (2.0 ** -10 + 8 * ez + 2.0 ** -17) * dz.abs()
    edz = es + U[dtype] * dz.abs()
    close(db, dz.sum(0), (es + (M + 32) * EPS32 * dz.abs()).sum(0) + U[dtype] * dz.sum(0).abs(), "db")
    for got, left, right, what in ((dw, dz.t(), X, "dw"), (dx, dz, W, "dx")):
        el = edz.t() if what == "dw" else edz
        want = left @ right
        bound = el @ right.abs() + (max(M, N) + 32) * EPS32 * (left.abs() @ right.abs()) + U[dtype] * want.abs()
        close(got, want, bound, what)


@gpu_only
@pytest.mark.parametrize("M", [7, 130])
@pytest.mark.parametrize("name", ["none", "gelu", "silu"])
def test_gradients_against_differences(gpu, M, name):
    x, w, b, r, dy = inputs(gpu, M, 40, 50, torch.float32)
    f = lambda *a: (void_amd.fused_linear(a[0], a[1], a[2], name, a[3]).double() * dy.double()).sum()
    args = [t.detach().requires_grad_() for t in (x, w, b, r)]
    grads = torch.autograd.grad(void_amd.fused_linear(args[0], args[1], args[2], name, args[3]), args, dy)
    for i in range(4):
        d = torch.randn_like(args[i])
        h = 2.0 ** -7
        up, down = [a.detach() for a in args], [a.detach() for a in args]
        up[i], down[i] = args[i].detach() + h * d, args[i].detach() - h * d
        slope = (f(*up) - f(*down)) / (2 * h)
        want = (grads[i].double() * d.double()).sum()
        # dZ along d, cubed, is what the truncation goes with; results are 2^-20 apart.
        dz = d.double() @ w.double().t() if i == 0 else x.double() @ d.double().t() if i == 1 else d.double()
        bound = (dy.double().abs() * (h * h * dz.abs() ** 3 + 2.0 ** -20 * (dz.abs() + 8) / h)).sum()
        assert (slope - want).abs() <= bound


@gpu_only
def test_streams_repeats_and_partial_gradients(gpu):
    x, w, b, r, dy = inputs(gpu, 300, 260, 2000, torch.bfloat16)
    a = [t.detach().requires_grad_() for t in (x, w, b, r)]
    call = lambda: torch.autograd.grad(void_amd.fused_linear(a[0], a[1], a[2], "gelu", a[3]), a, dy)
    first = call()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = call()
    s.synchronize()
    for p, q in zip(first, again):
        assert torch.equal(p, q)
    for i in range(4):
        c = [t.detach() for t in (x, w, b, r)]
        c[i].requires_grad_()
        g, = torch.autograd.grad(void_amd.fused_linear(c[0], c[1], c[2], "gelu", c[3]), c[i], dy)
        assert torch.equal(g, first[i])
    m = void_amd.FusedLinear(2000, 260, "gelu", dtype=torch.bfloat16, device=gpu)
    assert torch.equal(m(x, r), void_amd.fused_linear(x, m.weight, m.bias, "gelu", r))
    assert set(m.state_dict()) == {"weight", "bias"}


@gpu_only
@pytest.mark.parametrize("M,K", [(8, 4096), (300, 14000), (2048, 512)])
def test_graph_replays(gpu, M, K):
    x, w, b, r, _ = inputs(gpu, M, 384, K, torch.bfloat16)
    want = void_amd.fused_linear(x, w, b, "gelu", r)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = void_amd.fused_linear(x, w, b, "gelu", r)
    for _ in range(3):
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        assert torch.equal(void_amd.fused_linear(x, w, b, "gelu", r), want)


@gpu_only
def test_forward_mode_and_second_derivatives_are_refused(gpu):
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.randn(4, 16, device=gpu), torch.ones(4, 16, device=gpu))
        with pytest.raises((RuntimeError, NotImplementedError)):
            void_amd.fused_linear(x, torch.randn(8, 16, device=gpu))
    x = torch.randn(4, 16, device=gpu, requires_grad=True)
    g, = torch.autograd.grad(void_amd.fused_linear(x, torch.randn(8, 16, device=gpu)).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@gpu_only
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(1, 40, 5), (1, 9001, 131), (7, 100, 1001), (30, 33, 515), (64, 8193, 257), (50, 40, 4097)])
@pytest.mark.parametrize("shift,gap", [(1, 0), (1, 1), (2, 3)])
def test_rows_between_dwords(gpu, dtype, M, N, K, shift, gap):
    # What lies beside the rows is never seen.
    x, w, b, r, dy = inputs(gpu, M, N, K, dtype, M + N + K)

    def spread(t):
        rows, cols = t.shape
        buf = torch.full((rows * (cols + gap) + 8,), float("nan"), device=gpu, dtype=dtype)
        return buf[shift:shift + rows * (cols + gap)].view(rows, cols + gap)[:, :cols].copy_(t)
    check(spread(x), spread(w), b, spread(r), spread(dy), "silu")
    check(x, spread(w), b, None, spread(dy), "gelu")


@gpu_only
def test_offsets_past_31_bits(gpu):
    # A long X, whose gradient and whose product with dZ pass them; a long Y, slope and residual.
    x, w, b, _, _ = inputs(gpu, 128, 64, 4096, torch.bfloat16)
    M = (1 << 31) // 4096 + 40
    x = x.repeat(-(-M // 128), 1)[:M].requires_grad_()
    w.requires_grad_()
    y = void_amd.fused_linear(x, w, b)
    dy = torch.zeros_like(y)
    dy[-70:] = torch.randn(70, 64, device=gpu).to(y.dtype)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    tail = x.detach()[-70:], w.detach()
    want, bound = reference(*tail, b, None, dy[-70:], "none")
    close(y.detach()[-70:], want[0], bound[0], "y")
    close(dx[-70:], want[1], bound[1], "dx")
    close(dw, want[2], bound[2], "dw")  # rows of zeros add nothing
    assert not dx[:-70].any()
    del x, y, dy, dx, dw
    x, w, b, _, _ = inputs(gpu, 128, 8192, 64, torch.bfloat16)
    M = (1 << 31) // 8192 + 40
    x = x.repeat(-(-M // 128), 1)[:M].requires_grad_()
    r = torch.randn(64, 8192, device=gpu, dtype=torch.bfloat16).repeat(-(-M // 64), 1)[:M]
    y = void_amd.fused_linear(x, w, b, "silu", r)
    dx, = torch.autograd.grad(y, x, r)
    want, bound = reference(x.detach()[-70:], w, b, r[-70:], r[-70:], "silu")
    close(y.detach()[-70:], want[0], bound[0], "y")
    close(dx[-70:], want[1], bound[1], "dx")


@gpu_only
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M", [1, 8, 40, 100, 300])
def test_rows_far_apart(gpu, dtype, M):
    # The last token of each of M sequences: 256 rows (or all) span more than 2 GiB, where
    # 31-bit offsets end.  So do a weight's and a gradient's rows.  NaN lies between.
    N, K = 48, 72

    def far(t):
        rows, cols = t.shape
        pitch = (1 << 31) // t.element_size() // min(max(rows, 2), 256) // 64 * 64 + 64
        buf = torch.full((rows, pitch), float("nan"), dtype=dtype, device=gpu)
        buf[:, pitch - cols:] = t
        return buf[:, pitch - cols:]

    x, w, b, r, dy = inputs(gpu, M, N, K, dtype, M)
    check(far(x), w, b, far(r), dy, "gelu")
    check(x, w, b, None, far(dy), "none")
    check(x, far(w), b, r, far(dy), "silu")


@gpu_only
def test_one_row_of_any_pitch(gpu):
    # x and the gradient of one row: their pitch is never used.
    x, w, b, r, dy = inputs(gpu, 1, 40, 64, torch.bfloat16)
    place = lambda t: t.as_strided(t.shape, (1 << 33, 1))
    check(place(x), w, b, place(r), place(dy), "none")
    check(place(x), w, b, None, place(dy), "silu")
    # A weight of one row.
    x, w, b, r, dy = inputs(gpu, 100, 1, 64, torch.bfloat16)
    check(x, place(w), b, r, dy, "gelu")


@gpu_only
def test_more_columns_than_one_grid_axis_holds(gpu):
    # 2^24 groups of 16 rows of W, and of 64 columns' sums: more than 2^32 threads along one axis.
    N, K = (1 << 28) + 37, 2
    w = torch.randn(N, K, device=gpu, dtype=torch.bfloat16)
    b = torch.randn(N, device=gpu, dtype=torch.bfloat16).requires_grad_()
    x, dy = torch.randn(1, K, device=gpu).to(w.dtype), torch.randn(1, N, device=gpu, dtype=w.dtype)
    y = void_amd.fused_linear(x, w, b, "gelu")
    db, = torch.autograd.grad(y, b, dy)
    for part in (slice(0, 70), slice((1 << 27) - 40, (1 << 27) + 40), slice(N - 70, N)):
        want, bound = reference(x, w[part], b.detach()[part], None, dy[:, part], "gelu")
        close(y.detach()[:, part], want[0], bound[0], "y")
        close(db[part], want[3], bound[3] + U[b.dtype] * want[3].abs(), "db")


@gpu_only
def test_more_tiles_than_one_grid_axis_holds(gpu):
    # 2^24 tiles of 64 rows: more than 2^32 threads along one axis.
    M, N, K = (1 << 30) + 40, 3, 8
    g, w, b, _, _ = inputs(gpu, 1000, N, K, torch.bfloat16)
    x = g.repeat(-(-M // 1000), 1)[:M]
    y = void_amd.fused_linear(x, w, b, "silu")
    for part in (slice(0, 90), slice((1 << 29) - 40, (1 << 29) + 40), slice(M - 90, M)):
        want, bound = reference(x[part], w, b, None, None, "silu")
        close(y[part], want[0], bound[0], "y")


def test_refusals():
    x, w = torch.randn(2, 8), torch.randn(4, 8)
    f = void_amd.fused_linear
    with pytest.raises(RuntimeError, match="GPU"):
        f(x, w)
    for bad in ((x, w[:, :7]), (x, w[0]), (torch.tensor(1.0), w), (x, w, torch.zeros(3)), (x, w, torch.zeros(4, 1)),
                (x, w, None, "none", torch.zeros(2, 3)), (x, w, None, "none", torch.zeros(4)), (x, w, None, "softplus")):
        with pytest.raises(ValueError):
            f(*bad)
    for bad in ((x.double(), w.double()), (x, w.half()), (x, w, torch.zeros(4, dtype=torch.int32)),
                (x, w, None, "none", torch.zeros(2, 4).half())):
        with pytest.raises(TypeError):
            f(*bad)
    with pytest.raises(NotImplementedError):
        f(x, w, None, "tanh")
    with pytest.raises(ValueError):
        void_amd.FusedLinear(8, 4, "softplus")


def test_abi_refusals():
    import ctypes
    from void_amd import _lib
    lib = _lib.lib()
    at = 1 << 20  # a non-null, aligned address that is never read: every call below is refused
    base = dict(x=at, ldx=64, w=at, ldw=64, y=at, ldy=40, M=100, N=40, K=64, dtype=1, bias_dtype=1)
    for bad, code in ((dict(M=-1), -1), (dict(x=None), -1), (dict(y=None), -1), (dict(dtype=3), -2), (dict(ldx=63), -1),
                      (dict(ldy=39), -1), (dict(ldx=65), -2), (dict(K=63), -2), (dict(x=at + 2), -2), (dict(x=at + 1), -1),
                      (dict(activation=4), -2), (dict(slope=at), -1), (dict(bias=at, bias_dtype=2), -2),
                      (dict(N=1 << 31), -2), (dict(K=4096, ldx=4096, ldw=4096), -4)):
        a = _lib.LinearArgs(**{**base, **bad})
        assert lib.void_linear(ctypes.byref(a), None) == code, bad
    assert lib.void_linear_any_alignment(64) == 1 and lib.void_linear_any_alignment(65) == 0
    assert lib.void_linear_grad_x(at, 40, at, 64, 100, 40, 64, 1, at, 63, None, 0, None) == -1
    assert lib.void_linear_grad_x(at, 41, at, 64, 100, 40, 64, 1, at, 64, None, 0, None) == -2
    assert lib.void_linear_grad_w(at, 40, at, 60, 100, 40, 64, 1, at, 64, None, 0, None) == -2
    assert lib.void_linear_grad_z(at, 40, None, 100, 40, 1, at, 40, None, 1, None, 0, None) == -1
    assert lib.void_linear_grad_z(at, 40, None, 100, 40, 1, None, 0, at, 1, None, 0, None) == -4


def test_abi_refuses_rows_out_of_reach():
    import ctypes
    from void_amd import _lib
    lib = _lib.lib()
    at = 1 << 20  # never read
    base = dict(x=at, ldx=64, w=at, ldw=64, y=at, ldy=40, M=100, N=40, K=64, dtype=1, bias_dtype=1)
    for bad in (dict(ldx=1 << 24), dict(ldw=1 << 25)):
        a = _lib.LinearArgs(**{**base, **bad})
        assert lib.void_linear(ctypes.byref(a), None) == -2, bad
    assert lib.void_linear_grad_x(at, 1 << 24, at, 64, 100, 40, 64, 1, at, 64, None, 0, None) == -2
    assert lib.void_linear_grad_x(at, 40, at, 1 << 26, 100, 40, 64, 1, at, 64, None, 0, None) == -2
    assert lib.void_linear_grad_w(at, 1 << 25, at, 64, 100, 40, 64, 1, at, 64, None, 0, None) == -2
    assert lib.void_linear_grad_w(at, 40, at, 1 << 26, 100, 40, 64, 1, at, 64, None, 0, None) == -2
