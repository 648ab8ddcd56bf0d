"""The layers in front of the document head where they can go wrong: operands that lie in memory in unlike ways, infinities and values beyond the
type, rows far from zero, relu near its kink, long sums, what is kept, calls side by side.

Bounds as in test_gpu_token_layers: every rounding counted at its most."""

import pytest
import torch

from test_gpu_token_layers import ACTS, BF16, E, FP16, FP32, floor, linear_case, near, product, rand, unit

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------- operands that lie in memory in unlike ways
@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("m, k, f", [(300, 1, 200), (5, 1, 200), (2000, 1, 40), (300, 24, 200), (700, 1, 1)])
def test_gated_weights_of_differing_strides(dt, m, k, f):
    """With one input feature a contiguous weight has its features next to one another, a slice of a wider one has not."""
    from late_interaction_kernels_b200.token_layers import gated_feed_forward

    o = 16
    x, dy = rand(m, k, dt=dt), rand(m, o, dt=dt)
    plain, wide, across = rand(f, k, dt=dt), rand(f, k + 4, dt=dt)[:, 2 : 2 + k], rand(k, f, dt=dt).t()
    down, down_wide, down_across = rand(o, f, dt=dt), rand(o, 2 * f + 1, dt=dt)[:, f + 1 :], rand(f, o, dt=dt).t()
    for wg, wu, wd in ((plain, wide, down), (wide, plain, down_wide), (across, wide, down_across), (wide, across, down), (plain, across, down_wide)):
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu, wd)]
        y = gated_feed_forward(*leaves, activation=None)
        dx, dg_w, du_w, dd_w = torch.autograd.grad(y, leaves, dy)
        X, G, U, D, d = (t.double() for t in (x, wg, wu, wd, dy))
        g, u, dh = X @ G.t(), X @ U.t(), d @ D
        gs, us, dhs = X.abs() @ G.abs().t(), X.abs() @ U.abs().t(), d.abs() @ D.abs()
        # a factor is rounded, and its product with dh; products of k, o, f and m terms, the magnitudes of sums in place of the sums; a rounding
        # among subnormal numbers is off by `low`, the factor's times dh
        rel, low = 3 * unit(dt) + 4 * (k + o + f + m) * E, floor(dt) * (dhs + 1)
        near(y.detach(), (g * u) @ D.t(), (rel * gs * us + floor(dt)) @ D.abs().t(), "y")
        near(dx, (dh * u) @ G + (dh * g) @ U, (rel * dhs * us + low) @ G.abs() + (rel * dhs * gs + low) @ U.abs(), "dx")
        near(dg_w, (dh * u).t() @ X, (rel * dhs * us + low).t() @ X.abs(), "dw_gate")
        near(du_w, (dh * g).t() @ X, (rel * dhs * gs + low).t() @ X.abs(), "dw_up")
        near(dd_w, d.t() @ (g * u), d.abs().t() @ (rel * gs * us + floor(dt)), "dw_down")


# ----------------------------------------------------------------------------- infinities, and values beyond the type
# rows, features in and out: few rows, few rows of odd width, single CTAs, pairs, a product that is cut along k
KERNELS = [(3, 64, 72), (3, 63, 71), (300, 64, 72), (300, 63, 71), (9000, 64, 520), (300, 4000, 264)]


@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("m, k, n", KERNELS)
def test_activations_of_infinity(dt, m, k, n):
    from late_interaction_kernels_b200.token_layers import gated_feed_forward, linear

    inf = float("inf")
    x, w, b = rand(m, k, dt=dt), rand(n, k, dt=dt, scale=k**-0.5), torch.zeros(n, device="cuda", dtype=dt)
    b[1], b[n - 2] = inf, -inf
    ones, up = torch.zeros_like(w), torch.ones(n, device="cuda", dtype=dt)
    down = torch.zeros(2, n, device="cuda", dtype=dt)
    for act in ACTS[1:]:
        y = linear(x, w, b, activation=act)
        assert (y[:, 1] == (1 if act in ("tanh", "sigmoid") else inf)).all(), act
        if act in ("relu", "tanh", "sigmoid"):
            assert (y[:, n - 2] == (-1 if act == "tanh" else 0)).all(), act
        rest = [i for i in range(n) if i not in (1, n - 2)]
        assert torch.equal(y[:, rest], linear(x, w, torch.zeros_like(b), activation=act)[:, rest])
        bg = b.clone()
        bg[n - 2] = 0
        down[:, 1] = 1
        h = gated_feed_forward(x, w, ones, down[:, :n], b_gate=bg, b_up=up, activation=act)
        if act not in ("tanh", "sigmoid") and dt != FP32:  # (an fp32 infinity gives NaN or infinities in the second product)
            assert not torch.isfinite(h).any() and not torch.isfinite(h[:, 0]).any()


def same_kind(got, want):
    """NaN, infinities of either sign and finite numbers in the same places."""
    want = want.to(torch.float64)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isposinf(got), torch.isposinf(want)) and torch.equal(torch.isneginf(got), torch.isneginf(want))


@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("m, k, n", KERNELS)
def test_infinite_operands(dt, m, k, n):
    """An infinity gives infinities of its factors' signs, NaN where it meets 0 or another of the other sign, in every kernel and direction."""
    from late_interaction_kernels_b200.token_layers import linear

    inf = float("inf")
    x, w, dy = rand(m, k, dt=dt), rand(n, k, dt=dt), rand(m, n, dt=dt)
    x[0, 3], x[1, 5], x[1, 7], x[2, k - 1] = inf, -inf, inf, inf
    w[4, 3], w[5, 9], w[6, k - 1], w[7, 3] = -inf, inf, inf, 0
    dy[2, 8], dy[m - 1, 0] = -inf, inf
    x, w = x.requires_grad_(), w.requires_grad_()
    y = linear(x, w)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    X, W, D = x.detach().double(), w.detach().double(), dy.double()
    for got, want in ((y.detach(), X @ W.t()), (dx, D @ W), (dw, D.t() @ X)):
        same_kind(got, want)


@pytest.mark.parametrize("dt", [BF16, FP32])
@pytest.mark.parametrize("m", [3, 300, 9000])
def test_slopes_of_large_values(dt, m):
    """Far from zero a slope is 0 or 1, up to the largest finite value; at -50, the nearest, silu's is off by 49 exp(-50) = 9.5e-21."""
    from late_interaction_kernels_b200.token_layers import gated_feed_forward, linear

    n = 64
    mags = torch.tensor([50.0, 1e4, 1e8, 1e12, 2e13, 1e16, 1e20, 1e30], device="cuda").repeat(n // 8)
    z = (mags * torch.where(torch.rand(m, n, device="cuda") < 0.5, -1.0, 1.0)).to(dt)
    dy = rand(m, n, dt=dt)
    eye = torch.eye(n, device="cuda", dtype=dt)
    one = torch.ones(n, device="cuda", dtype=dt)
    for act in ACTS[1:]:
        want = dy * (z > 0) if act not in ("tanh", "sigmoid") else torch.zeros_like(dy)
        x = z.clone().requires_grad_()
        (dx,) = torch.autograd.grad(linear(x, eye, activation=act), [x], dy)
        assert ((dx - want).abs() <= 1e-20 * dy.abs()).all(), act
        x = z.clone().requires_grad_()
        (dx,) = torch.autograd.grad(gated_feed_forward(x, eye, torch.zeros_like(eye), eye, b_up=one, activation=act), [x], dy)
        assert ((dx - want).abs() <= 1e-20 * dy.abs()).all(), act


@pytest.mark.parametrize("dt", [FP16, BF16, FP32])
@pytest.mark.parametrize("m, k, n", KERNELS)
def test_slopes_where_what_is_kept_is_beyond_its_type(dt, m, k, n):
    """z of +-131072 is finite in the sums and the result, +-infinity where it is kept in fp16; its slope is 0 or 1 all the same."""
    from late_interaction_kernels_b200.token_layers import linear

    x, w = rand(m, k, dt=dt, scale=0.1), rand(n, k, dt=dt, scale=0.1)
    x[:, 0] = 256
    w[:, 0] = torch.where(torch.rand(n, device="cuda") < 0.5, -512.0, 512.0).to(dt)
    dy = rand(m, n, dt=dt, scale=2.0**-6)
    b = torch.zeros(n, device="cuda", dtype=dt)
    for act in ACTS[1:]:
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        y = linear(*leaves, activation=act)
        dx, dw, db = torch.autograd.grad(y, leaves, dy)
        open_ = (w[:, 0] > 0).double() if act not in ("tanh", "sigmoid") else torch.zeros(n, device="cuda", dtype=torch.float64)
        assert torch.isfinite(y[:, w[:, 0] < 0]).all(), act
        dz = dy.double() * open_
        for got, (want, err), name in ((dx, product(dz, w.double().t()), "dx"), (dw, product(dz.t(), x.double().t()), "dw")):
            near(got, want, err, f"{act} {name}")
        near(db, dz.sum(0), 2 * m * E * dz.abs().sum(0), f"{act} db")


# ----------------------------------------------------------------------------- rows far from zero
FAR_WIDTHS = [7, 100, 300, 768, 1000, 1001, 1023, 1500, 3000, 5000, 9001, 16385, 20000]


@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("width", FAR_WIDTHS)
def test_layer_norm_of_constant_rows(dt, width):
    """A row of one value is its own mean: what is left is zero, whatever the width's reciprocal and the sum of the row round to."""
    from late_interaction_kernels_b200.token_layers import layer_norm

    values = torch.tensor([3.25, 7.0, 0.1, 100.0, 1000.0, 1001.0, -999.0, 0.0], device="cuda").to(dt)
    x = values[:, None].expand(8, width).contiguous().requires_grad_()
    y = layer_norm(x)
    # the mean is off by a rounding of its sum's steps, what corrects it by as much of that again
    steps = min(width, 64) + 16
    bound = (2 * steps * E) ** 2 * values.double().abs()[:, None] * 1e-5**-0.5
    near(y.detach(), torch.zeros(8, width, dtype=torch.float64, device="cuda"), bound.expand(8, width), "y")
    dy = rand(8, width, dt=dt)
    (dx,) = torch.autograd.grad(y, [x], dy)
    d = dy.double()
    # the mean that is kept is the value itself, or its nearest neighbour: h is at most a step of the value over the deviation
    h = 2 * E * values.double().abs()[:, None] * 1e-5**-0.5
    s = d.abs().mean(1, keepdim=True)
    near(dx, 1e-5**-0.5 * (d - d.mean(1, keepdim=True)), 1e-5**-0.5 * (8 * steps * E * (d.abs() + s) + h * h * s + 2 * h * h * (d.abs() + s)), "dx")


@pytest.mark.parametrize("dt", [BF16, FP32])
@pytest.mark.parametrize("width", FAR_WIDTHS)
def test_layer_norm_of_rows_beyond_the_squares_of_fp32(dt, width):
    """Squares of differences beyond 3e38 leave no deviation to divide by but infinity: the row is zeros, not NaN."""
    from late_interaction_kernels_b200.token_layers import layer_norm

    x = torch.tensor([1e30, -3e33, 7e25, 1e20], device="cuda").to(dt)[:, None].expand(4, width).contiguous()
    assert torch.isfinite(layer_norm(x)).all()
    assert torch.equal(layer_norm(rand(5, width, dt=dt) * 1e30), torch.zeros(5, width, device="cuda", dtype=dt))


@pytest.mark.parametrize("width", FAR_WIDTHS)
def test_layer_norm_far_from_zero(width):
    """fp32 rows whose mean is ten thousand times their deviation: the result is as near to 64 bits as that of rows around zero."""
    from late_interaction_kernels_b200.token_layers import layer_norm

    for shift in (1e4, -3e4):
        x = rand(9, width, dt=FP32, shift=shift)
        v = x.double()
        mean, var = v.mean(1, keepdim=True), v.var(1, correction=0, keepdim=True)
        hat = (v - mean) / (var + 1e-5).sqrt()
        steps = min(width, 64) + 16
        # differences from the rounded mean are exact to a rounding; their mean and that of their squares are sums of `steps`
        off = steps * E * (abs(shift) * E * steps / var.sqrt() + hat.abs().mean(1, keepdim=True))
        near(layer_norm(x), hat, off + hat.abs() * (2 * steps + 8) * E + 4 * E, "y")


# ----------------------------------------------------------------------------- relu near its kink
def cancelling(m, h, n, dt):
    """Rows and features whose products cancel to +-2^-20 in another order than they come in."""
    a, b = rand(m, h, dt=dt), rand(n, h, dt=dt)
    perm = torch.randperm(h, device="cuda")
    tiny = torch.where(torch.rand(m, 1, device="cuda") < 0.5, -1.0, 1.0) * 2.0**-10
    return torch.cat([a, a[:, perm], tiny.to(dt)], 1), torch.cat([b, -b[:, perm], torch.full((n, 1), 2.0**-10, device="cuda", dtype=dt)], 1)


@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("m, pad", [(3, 7), (3, 0), (40, 7), (700, 7), (700, 0), (5000, 7)])
@pytest.mark.parametrize("h", [496, 2000])
def test_relu_where_all_neighbours_are_near_its_kink(dt, m, pad, h):
    from late_interaction_kernels_b200.token_layers import gated_feed_forward, linear

    n = 200
    x, w = cancelling(m, h, n, dt)
    zero = lambda t: torch.cat([t, torch.zeros(t.shape[0], pad, device="cuda", dtype=dt)], 1)
    x, w = zero(x), zero(w)
    z = x.double() @ w.double().t()
    assert float((z.abs() - 2.0**-20).abs().max()) < 2.0**-30
    open_ = (z > 0).double()
    for bias in (None, torch.zeros(n, device="cuda", dtype=dt)):
        x1 = x.clone().requires_grad_()
        (dx,) = torch.autograd.grad(linear(x1, w, bias, activation="relu"), [x1], torch.ones(m, n, device="cuda", dtype=dt))
        near(dx, open_ @ w.double(), 2 * n * E * (open_ @ w.double().abs()), "dx")
    g1 = w.clone().requires_grad_()
    y = gated_feed_forward(x, g1, torch.zeros_like(w), torch.ones(8, n, device="cuda", dtype=dt), b_up=torch.ones(n, device="cuda", dtype=dt), activation="relu")
    (dg,) = torch.autograd.grad(y, [g1], torch.ones_like(y))
    near(dg, 8 * open_.t() @ x.double(), 2 * m * E * 8 * open_.t() @ x.double().abs(), "dw_gate")


@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("m", [3, 300, 9000])
def test_relu_beside_features_that_are_off_zero_or_infinite(dt, m):
    """One feature switched off by its bias, a dead one, one with an infinite weight and rows of padding: the others' gradients are as without."""
    from late_interaction_kernels_b200.token_layers import linear

    k, n = 128, 96
    x, w, b = rand(m, k, dt=dt), rand(n, k, dt=dt, scale=k**-0.5), rand(n, dt=dt)
    x[m // 2 :] = 0
    dy = rand(m, n, dt=dt)
    w[5], b[5] = 0, 0
    b[3], b[40] = -60000, 60000
    want = torch.where(z_of(x, w, b) > 0, dy.double(), 0)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(linear(*leaves, activation="relu"), leaves, dy)
    near(dx, want @ w.double(), 2 * n * E * want.abs() @ w.double().abs(), "dx")
    near(dw, want.t() @ x.double(), 2 * m * E * want.abs().t() @ x.double().abs(), "dw")
    near(db, want.sum(0), 2 * m * E * want.abs().sum(0), "db")
    leaves[1].data[60, 7] = float("inf")
    rest = [i for i in range(n) if i != 60]
    dw2 = torch.autograd.grad(linear(*leaves, activation="relu"), leaves, dy)[1]
    assert torch.equal(dw2[rest], dw[rest])


def z_of(x, w, b):
    return x.double() @ w.double().t() + b.double()


# ----------------------------------------------------------------------------- long sums
LONG = [(20000, 40, 24), (30000, 96, 200), (30001, 95, 200), (66011, 72, 40), (65600, 264, 520), (140000, 16, 8), (70001, 8, 300)]
LONG_K = [(700, 33000, 260), (5200, 17000, 1100), (40, 66000, 72), (2600, 70000, 264)]


@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("m, k, n", LONG)
def test_long_sums_of_whole_numbers_are_exact(dt, m, k, n):
    """Sums over many tokens whose every partial sum is a whole number below 2^24: in any order and with any adder of 24 bits they are exact, and a
    token, a slab or a share that is left out or taken twice shows."""
    from late_interaction_kernels_b200.token_layers import gated_feed_forward, linear

    ints = lambda *shape: torch.randint(-3, 4, shape, device="cuda").to(dt)
    x, dy = ints(m, k), ints(m, n)
    w, b = torch.zeros(n, k, device="cuda", dtype=FP32).requires_grad_(), torch.zeros(n, device="cuda", dtype=FP32).requires_grad_()
    dw, db = torch.autograd.grad(linear(x, w, b), [w, b], dy)
    assert dw.dtype == FP32 and torch.equal(dw.double(), dy.double().t() @ x.double()) and torch.equal(db.double(), dy.double().sum(0))
    # a gated block whose gate is 1 everywhere and whose up projection picks a feature of x: its factors and gradients are whole numbers of a few bits
    pick = torch.zeros(n, k, device="cuda", dtype=FP32)
    pick[torch.arange(n), torch.arange(n) % k] = 1
    pick.requires_grad_()
    wg, wd = torch.zeros(n, k, device="cuda", dtype=FP32).requires_grad_(), torch.zeros(8, n, device="cuda", dtype=FP32)
    wd[torch.arange(n) % 8, torch.arange(n)] = 1
    wd.requires_grad_()
    bg, d = torch.ones(n, device="cuda", dtype=FP32).requires_grad_(), ints(m, 8)
    got = torch.autograd.grad(gated_feed_forward(x, wg, pick, wd, b_gate=bg, activation=None), [wg, pick, wd, bg], d)
    X, u, dh = x.double(), x.double() @ pick.detach().double().t(), d.double() @ wd.detach().double()
    for g, want in zip(got, ((dh * u).t() @ X, dh.t() @ X, d.double().t() @ u, (dh * u).sum(0))):
        assert g.dtype == FP32 and torch.equal(g.double(), want)


@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("i", range(len(LONG_K)))
def test_linear_of_many_features(dt, i):
    """Products with a bias, an activation and a residual whose sums are cut for their length alone."""
    linear_case(*LONG_K[i], dt, ACTS[1 + i], True, True)


@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("n, k", [(1024, 1024), (4096, 1024), (128, 128)])
def test_fp32_gradients_of_many_tokens(dt, n, k):
    """Terms of one sign: an addition of 16 products cuts off up to four steps of what has been summed.  One accumulator goes over 8192 tokens at most:
    512 additions, with half of the whole sum on average, so 1024 steps of 2^-23 of the result."""
    from late_interaction_kernels_b200.token_layers import linear

    m = 65536
    x, dy = rand(m, k, dt=dt).abs() + 0.5, rand(m, n, dt=dt).abs() + 0.5
    w = torch.zeros(n, k, device="cuda", dtype=FP32).requires_grad_()
    (dw,) = torch.autograd.grad(linear(x, w), [w], dy)
    want = torch.zeros(n, k, device="cuda", dtype=torch.float64)
    for i in range(0, m, 8192):
        want += dy[i : i + 8192].double().t() @ x[i : i + 8192].double()
    assert float(((dw.double() - want).abs() / want).max()) < 1024 * 2.0**-23 + 16 * E


# ----------------------------------------------------------------------------- what is kept
def test_nothing_is_kept_for_gradients_that_are_made_of_dy_alone():
    """With everything frozen but a residual, or the bias behind a gated block's last product, the call holds its result and no more."""
    from late_interaction_kernels_b200.token_layers import gated_feed_forward, linear

    m, k, f = 4096, 256, 1024
    x, w, wg, wd, r, d = rand(m, k, dt=BF16), rand(k, k, dt=BF16), rand(f, k, dt=BF16), rand(k, f, dt=BF16), rand(m, k, dt=BF16), rand(m, k, dt=BF16)
    b = rand(k, dt=BF16)
    for fn in (lambda r, b: linear(x, w, activation="gelu", residual=r), lambda r, b: gated_feed_forward(x, wg, wg, wd, b_down=b, residual=r)):
        leaves = [t.clone().requires_grad_() for t in (r, b)]
        fn(*leaves)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = fn(*leaves)
        torch.cuda.synchronize()
        assert torch.cuda.memory_allocated() - before <= y.numel() * y.element_size() + 4096
        dr, db = torch.autograd.grad(y, leaves, d, allow_unused=True)
        assert torch.equal(dr, d)
        if db is not None:
            near(db, d.double().sum(0), 2 * m * E * d.double().abs().sum(0), "db_down")
        assert torch.equal(y, fn(*(t.detach() for t in leaves)))


# ----------------------------------------------------------------------------- captured, and beside another stream
@pytest.mark.parametrize("wdt", [BF16, FP32])
def test_relu_steps_in_two_graphs_and_on_two_streams(wdt):
    """The lengths for relu's kink and the shares of long sums are workspaces of a call's own."""
    from late_interaction_kernels_b200 import check_device_status
    from late_interaction_kernels_b200.token_layers import gated_feed_forward, linear

    k = 192
    data = [(rand(m, k, dt=BF16).requires_grad_(), rand(m, k, dt=BF16)) for m in (20000, 700)]
    p = [rand(*s, dt=wdt, scale=k**-0.5).requires_grad_() for s in ((k, k), (2 * k, k), (2 * k, k), (k, 2 * k))]

    def step(x, d):
        y = gated_feed_forward(linear(x, p[0], activation="relu", residual=x), *p[1:], activation="relu")
        return [y.detach(), *torch.autograd.grad(y, [x, *p], d)]

    want = [step(*d) for d in data]
    graphs = []
    for d in data:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*d)
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in data]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i][0].replay()
                got[i].append([t.clone() for t in graphs[i][1]])
                got[1 - i].append(step(*data[1 - i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            for a, b in zip(g, want[i]):
                assert torch.equal(a, b)
    check_device_status()
