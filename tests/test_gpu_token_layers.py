"""The layers in front of the document head against their definition in 64 bits.

Every comparison is element by element, against a bound that is the sum of what each rounding on the way can do at most.  With
u = eps / 2 of the type (a rounding's largest relative error), e = 2^-24 (fp32) and S the same sum with magnitudes:

  product         n terms added in fp32 in any order, by an adder that may truncate:     2 n e S
  activation      fp32 functions within a few steps (fp32), 2^-16 of the value's scale (16-bit types, far below their u)
  what is kept    z, and of a gated block u act'(g), act(g) and h, in the type: u of each; an error of z goes through the
                  activation's largest slope (1.13 for all of them) or curvature (at most 0.9)
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh", "tanh", "sigmoid"]
SLOPE, CURVE = 1.13, 0.9  # largest |act'| and |act''| (relu: its kink is not crossed, a rounding keeps the sign)
E = 2.0**-24


def unit(dt):
    return torch.finfo(dt).eps / 2


def floor(dt):
    """Half a step among the subnormal numbers, where a rounding's error is no longer relative."""
    return {BF16: 2.0**-134, FP16: 2.0**-25, FP32: 2.0**-150}[dt]


def act64(z, act):
    if act is None:
        return z
    if act == "gelu":
        return 0.5 * z * torch.special.erfc(-z * 0.5**0.5)  # (1 + erf would cancel in the lower tail, in 64 bits too)
    if act == "gelu_tanh":
        return z * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (z + 0.044715 * z**3))  # (1 + tanh(y)) / 2, which cancels as well
    return {"relu": torch.relu, "silu": torch.nn.functional.silu, "tanh": torch.tanh, "sigmoid": torch.sigmoid}[act](z)


def slope64(z, act):
    with torch.enable_grad():
        v = z.detach().clone().requires_grad_()
        return torch.autograd.grad(act64(v, act).sum(), v)[0]


def act_err(z, dt):
    """What the fp32 evaluation of an activation or its slope may be off, relative to |z| + 1."""
    return (z.abs() + 1) * (2.0**-20 if dt == FP32 else 2.0**-16)


def near(got, want, err, what):
    """|got - want| <= err, element by element, with rounding to got's type and 1 % for the terms of second order."""
    assert got.shape == want.shape and got.dtype in (BF16, FP16, FP32), what
    bound = 1.01 * (err + unit(got.dtype) * (want.abs() + err)) + floor(got.dtype)
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, the worst by {float((off / bound).nan_to_num(9e9).max()):.3g} bounds"


def rand(*shape, dt, scale=1.0, shift=0.0):
    return (torch.randn(*shape, device="cuda") * scale + shift).to(dt)


def mm(a, b):
    return a @ b


# ----------------------------------------------------------------------------- layer norm
WIDTHS = [1, 2, 3, 8, 17, 64, 100, 255, 256, 257, 512, 768, 1000, 1023, 1024, 1025, 2048, 2500, 4096, 4104, 5000, 8192, 9001, 16384]


def norm_bounds(x, w, b, dy, eps, dt):
    """The definition and what fp32 may be off: a row's mean within n e of its magnitudes, its deviation accordingly."""
    n = x.shape[1]
    mean = x.mean(1, keepdim=True)
    cen = x - mean
    var = cen.square().mean(1, keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    # sums over a row: at most 64 additions in one register after another, then pairwise
    steps = min(n, 64) + 16
    d_mean = steps * E * x.abs().mean(1, keepdim=True)
    d_cen = d_mean + E * cen.abs()
    hat = cen * rstd
    d_rstd = (steps * E + (d_mean * cen.abs().mean(1, keepdim=True) * 2 + d_mean**2) / (var + eps)) * 1.0
    d_hat = d_cen * rstd + hat.abs() * (d_rstd + 4 * E)
    W = torch.ones(n, dtype=torch.float64, device="cuda") if w is None else w
    B = torch.zeros(n, dtype=torch.float64, device="cuda") if b is None else b
    y = hat * W + B
    out = {"y": (y, d_hat * W.abs() + 2 * E * (hat * W).abs() + E * B.abs())}
    if dy is None:
        return out
    g = dy * W
    c1, c2 = g.mean(1, keepdim=True), (g * hat).mean(1, keepdim=True)
    d_c1 = (steps + 1) * E * g.abs().mean(1, keepdim=True)
    d_c2 = (g.abs() * (d_hat + (steps + 2) * E * hat.abs())).mean(1, keepdim=True)
    dx = rstd * (g - c1 - hat * c2)
    d_dx = rstd * (E * g.abs() + d_c1 + hat.abs() * d_c2 + d_hat * c2.abs()) + dx.abs() * (d_rstd + 4 * E) + rstd * 3 * E * (g.abs() + c1.abs() + (hat * c2).abs())
    m = x.shape[0] + 64
    out["dx"] = (dx, d_dx)
    out["dw"] = ((dy * hat).sum(0), (dy.abs() * (d_hat + m * E * hat.abs())).sum(0))
    out["db"] = (dy.sum(0), m * E * dy.abs().sum(0))
    return out


@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("width", WIDTHS)
def test_layer_norm(dt, width):
    from late_interaction_kernels_b200.token_layers import layer_norm

    rows = 1 if width == 17 else (7 if width > 4096 else 131)
    x = rand(rows, width, dt=dt, scale=2.0, shift=0.5).requires_grad_()
    w, b = rand(width, dt=dt, scale=0.3, shift=1.0).requires_grad_(), rand(width, dt=dt).requires_grad_()
    dy = rand(rows, width, dt=dt)
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    want = norm_bounds(x.detach().double(), w.detach().double(), b.detach().double(), dy.double(), 1e-5, dt)
    for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        near(got.detach(), *want[name], name)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b), y)


@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("which", ["none", "weight", "bias", "fp32", "mixed"])
def test_layer_norm_parameters(dt, which):
    from late_interaction_kernels_b200.token_layers import layer_norm

    x = rand(3, 5, 40, 768, dt=dt).requires_grad_()
    w = None if which in ("none", "bias") else rand(768, dt=FP32 if which in ("fp32", "mixed") else dt).requires_grad_()
    b = None if which in ("none", "weight") else rand(768, dt=FP32 if which == "fp32" else dt).requires_grad_()
    y = layer_norm(x, w, b, eps=1e-3)
    dy = rand(3, 5, 40, 768, dt=dt)
    leaves = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    flat = lambda t: None if t is None else t.detach().double().reshape(-1, 768) if t.dim() > 1 else t.detach().double()
    want = norm_bounds(flat(x), flat(w), flat(b), flat(dy), 1e-3, dt)
    near(y.detach().reshape(-1, 768), *want["y"], "y")
    for t, g, name in zip(leaves, grads, ["dx"] + (["dw"] if w is not None else []) + (["db"] if b is not None else [])):
        assert g.dtype == t.dtype and g.shape == t.shape
        near(g.reshape(-1, 768) if name == "dx" else g, *want[name], name)


@pytest.mark.parametrize("rows", [0, 1, 2, 295, 296, 297, 5000, 40001])
def test_layer_norm_row_counts(rows):
    from late_interaction_kernels_b200.token_layers import layer_norm

    x, w, b = rand(rows, 256, dt=BF16).requires_grad_(), rand(256, dt=BF16).requires_grad_(), rand(256, dt=BF16).requires_grad_()
    dy = rand(rows, 256, dt=BF16)
    y = layer_norm(x, w, b)
    got = torch.autograd.grad(y, (x, w, b), dy)
    want = norm_bounds(x.detach().double(), w.detach().double(), b.detach().double(), dy.double(), 1e-5, BF16)
    near(y.detach(), *want["y"], "y")
    for g, n in zip(got, ("dx", "dw", "db")):
        near(g, *want[n], n)


def test_layer_norm_strides_and_constant_rows():
    from late_interaction_kernels_b200.token_layers import layer_norm

    big = rand(64, 1600, dt=BF16)
    for x in (big[:, :768], big[:, 5:773], big[:, ::2], big.t()[:768].t(), big[:1, :768].expand(9, 768), big[::3, 100:868]):
        y = layer_norm(x)
        near(y, *norm_bounds(x.double(), None, None, None, 1e-5, BF16)["y"], "y")
        assert torch.equal(y, layer_norm(x.contiguous()))
    # a row of one value has no deviation: zeros times the weight, plus the bias; eps alone keeps the gradient finite
    x = torch.full((4, 300), 3.25, device="cuda", dtype=FP16).requires_grad_()
    b = rand(300, dt=FP16)
    y = layer_norm(x, None, b)
    assert torch.equal(y.detach(), b.expand(4, 300))
    y.float().sum().backward()
    assert torch.isfinite(x.grad).all()
    # infinities and NaN stay in their rows
    x = rand(6, 512, dt=FP32)
    x[1, 3], x[4, 500] = float("inf"), float("nan")
    y = layer_norm(x)
    assert torch.isnan(y[[1, 4]]).all() and torch.isfinite(y[[0, 2, 3, 5]]).all()


# ----------------------------------------------------------------------------- linear
def product(a, b):
    """a @ b.T in 64 bits and what n additions in fp32 may be off."""
    return mm(a, b.t()), 2 * a.shape[1] * E * mm(a.abs(), b.abs().t())


def check_linear(x, w, b, r, dy, act, y, grads, dt):
    x, w, dy = x.detach().double(), w.detach().double().to(dt).double(), dy.double()
    z, dz_err = product(x, w)
    if b is not None:
        z = z + b.detach().double().to(dt).double()
        dz_err = dz_err + E * z.abs()
    y64, y_err = act64(z, act), SLOPE * dz_err + (act_err(z, dt) if act else 0)
    if r is not None:
        y64 = y64 + r.detach().double()
        y_err = y_err + E * y64.abs()
    near(y.detach(), y64, y_err, "y")
    u = unit(dt)
    dz = dy * slope64(z, act)
    # z is kept rounded; dz is rounded before the products
    err = dy.abs() * (CURVE * (u * (z.abs() + dz_err) + dz_err + floor(dt)) + act_err(z, dt)) if act and act != "relu" else torch.zeros_like(dz)
    if act == "relu":
        err = torch.where(z.abs() <= dz_err + floor(dt), dy.abs(), err)  # the kink: either side
    if act:
        err = err + u * (dz.abs() + err) + floor(dt)
    dx, dx_err = product(dz, w.t())
    near(grads["x"], dx, dx_err + mm(err, w.abs()), "dx")
    dw, dw_err = product(dz.t(), x.t())
    near(grads["w"], dw, dw_err + mm(err.t(), x.abs()), "dw")
    if b is not None:
        m = dz.shape[0]
        near(grads["b"], dz.sum(0), err.sum(0) + 2 * m * E * dz.abs().sum(0), "db")
    if r is not None:
        assert torch.equal(grads["r"], dy.to(dt))


def linear_case(m, k, n, dt, act, bias, residual, wdt=None):
    from late_interaction_kernels_b200.token_layers import linear

    x = rand(m, k, dt=dt).requires_grad_()
    w = rand(n, k, dt=wdt or dt, scale=1.5 * k**-0.5).requires_grad_()
    b = rand(n, dt=wdt or dt).requires_grad_() if bias else None
    r = rand(m, n, dt=dt).requires_grad_() if residual else None
    y = linear(x, w, b, activation=act, residual=r)
    assert y.shape == (m, n) and y.dtype == dt
    dy = rand(m, n, dt=dt)
    named = [(s, t) for s, t in (("x", x), ("w", w), ("b", b), ("r", r)) if t is not None]
    grads = dict(zip([s for s, _ in named], torch.autograd.grad(y, [t for _, t in named], dy)))
    for s, t in named:
        assert grads[s].dtype == t.dtype and grads[s].shape == t.shape
    check_linear(x, w, b, r, dy, act, y, grads, dt)
    with torch.no_grad():
        assert torch.equal(linear(x, w, b, activation=act, residual=r), y)


SHAPES = [(1, 1, 1), (1, 7, 3), (2, 64, 5), (5, 16, 16), (8, 768, 768), (9, 768, 130), (16, 512, 1024), (17, 512, 1000), (32, 768, 128), (33, 100, 65), (64, 72, 264),
          (128, 128, 128), (129, 255, 257), (255, 264, 248), (300, 768, 520), (700, 1001, 333), (2050, 192, 72), (4096, 64, 64), (20000, 40, 24), (1000, 2048, 136),
          (2500, 520, 392), (4100, 260, 1030), (30000, 96, 200), (40, 1, 1), (300, 1, 5), (5, 300, 1),
          (300, 4000, 260), (128, 2900, 70), (3000, 2700, 300), (700, 640, 1600), (200, 1500, 136), (16, 5200, 24), (6, 12300, 40)]


@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_linear_shapes(dt, i):
    linear_case(*SHAPES[i], dt, ACTS[i % 7], i % 3 != 0, i % 2 == 0)


@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [3, 40, 515])
def test_linear_activations(dt, act, m):
    linear_case(m, 256, 320, dt, act, True, True)


@pytest.mark.parametrize("dt", [BF16, FP16])
def test_linear_fp32_parameters(dt):
    linear_case(150, 320, 200, dt, "gelu", True, True, wdt=FP32)
    linear_case(3, 320, 200, dt, None, True, False, wdt=FP32)


def test_activations_over_their_range():
    """The identity as weights: what comes out is the activation, for values from subnormal ones to where it saturates."""
    from late_interaction_kernels_b200.token_layers import linear

    mags = torch.cat([torch.logspace(-30, 1.5, 2000), torch.linspace(0, 14, 2096)])
    z = torch.cat([-mags, mags]).cuda().reshape(-1, 64)
    for dt in (BF16, FP16, FP32):
        x, w = z.to(dt), torch.eye(64, device="cuda", dtype=dt)
        for act in ACTS[1:]:
            want = act64(x.double(), act)
            got = linear(x, w, activation=act).double()
            # relative to the value itself: half a step and the fit's error, and what the exponential makes of its rounded argument.
            # exp(-v) with v off by d is off by |d| relative to itself; v (z^2 / 2; twice gelu_tanh's y; z or 2 z) is a product of
            # up to three fp32 factors, one of them a rounded constant: |d| <= 4 e |v| = 2^-22 |v|.  Where exp underflows in fp32,
            # values of 2^-120 may be lost.
            q = x.double()
            v = {"gelu": q * q, "gelu_tanh": 1.6 * (q + 0.044715 * q**3)}.get(act, 2 * q).abs()
            rel = unit(dt) + (2.0**-16 if dt != FP32 else 2.0**-19) + 2.0**-22 * v
            off = (got - want).abs() - rel * want.abs() - floor(dt) - 2.0**-118
            assert (off <= 0).all(), (dt, act, float(x.flatten()[off.argmax()]), float(off.max()))


@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("m", [3, 40, 700, 5000])
def test_relu_near_its_kink(dt, m):
    """z that is next to nothing beside the products that it is a sum of, as sums that cut off what they shift out get wrong: half the products
    cancel the other half (in another order, so that partial sums are large), what is left is +-2^-20, and the slope is its sign."""
    from late_interaction_kernels_b200.token_layers import gated_feed_forward, linear

    h, n = 496, 200
    a, b = rand(m, h, dt=dt), rand(n, h, dt=dt)
    perm = torch.randperm(h, device="cuda")
    tiny = torch.where(torch.rand(m, 1, device="cuda") < 0.5, -1.0, 1.0) * 2.0**-10
    x = torch.cat([a, a[:, perm], tiny.to(dt).expand(m, 8)], 1)
    w = torch.cat([b, -b[:, perm], torch.full((n, 8), 2.0**-13, device="cuda").to(dt)], 1)
    big = rand(n, x.shape[1], dt=dt)  # (neighbours of the usual size)
    w[::2] = big[::2]
    bias = torch.zeros(n, device="cuda", dtype=dt)
    for bi in (None, bias):
        x1 = x.clone().requires_grad_()
        y = linear(x1, w, bi, activation="relu")
        (dx,) = torch.autograd.grad(y, [x1], torch.ones_like(y))
        z = x.double() @ w.double().t()
        assert float(z[:, 1::2].abs().max()) == 2.0**-20
        want = (z > 0).double() @ w.double()
        near(dx, want, 2 * n * E * ((z > 0).double() @ w.double().abs()), "dx")
    # the gate of a block: only odd features get through to the result, as 1 where the gate is open
    wd = torch.zeros(8, n, device="cuda", dtype=dt)
    wd[:, 1::2] = 1
    up = torch.zeros_like(w)
    up1 = torch.ones(n, device="cuda", dtype=dt)
    x1 = x.clone().requires_grad_()
    g1 = w.clone().requires_grad_()
    y = gated_feed_forward(x1, g1, up, wd, b_up=up1, activation="relu")
    (dg,) = torch.autograd.grad(y, [g1], torch.ones_like(y))
    open_ = (z[:, 1::2] > 0).double()
    near(dg[1::2], 8 * open_.t() @ x.double(), 2 * m * E * 8 * open_.t() @ x.double().abs(), "dw_gate")


def test_linear_strides():
    """Rows that do not follow one another, start off 16 bytes, overlap or lie across: the kernels differ, the numbers are held to the same bounds."""
    from late_interaction_kernels_b200.token_layers import linear

    big, W = rand(40, 40, 512, dt=BF16), rand(96, 512, dt=BF16)
    base = rand(40, 40, 97, dt=BF16)
    for x in (big[..., :256], big[..., 1:257], big[::2, :, 256:], big[..., ::2], big.transpose(0, 1)[..., :256], big[:1, :1, :256].expand(3, 5, 256)):
        for w in (W[:, :256], W[:, 3:259], W[:, ::2], W.t().contiguous().t()[:, :256]):
            for r in (base[: x.shape[0], : x.shape[1], :96], base[: x.shape[0], : x.shape[1], 1:]):
                leaves = [t.detach().requires_grad_() for t in (x, w, r)]
                y = linear(leaves[0], leaves[1], activation="silu", residual=leaves[2])
                dy = rand(1, 1, 96, dt=BF16).expand(y.shape)  # a broadcast gradient, rows that overlap
                grads = dict(zip("xwr", torch.autograd.grad(y, leaves, dy)))
                flat = lambda t: t.reshape(-1, t.shape[-1])
                check_linear(flat(x), w, None, flat(r), flat(dy), "silu", flat(y), {"x": flat(grads["x"]), "w": grads["w"], "r": flat(grads["r"])}, BF16)


def test_linear_nan_and_infinity_stay_in_their_rows():
    from late_interaction_kernels_b200.token_layers import linear

    for dt in (BF16, FP32):
        for m in (4, 300):
            x, w = rand(m, 128, dt=dt), rand(64, 128, dt=dt)
            x[1, 5], x[2, 100] = float("nan"), float("inf")
            y = linear(x, w, activation="gelu")
            keep = [0] + list(range(3, m))
            assert torch.isnan(y[1]).all() and not torch.isfinite(y[2]).all() and torch.isfinite(y[keep]).all()
            assert torch.equal(y[keep], linear(x.nan_to_num(0, 0, 0), w, activation="gelu")[keep])


# ----------------------------------------------------------------------------- gated feed-forward
def gated_case(m, k, f, o, dt, act, bias, residual, wdt=None):
    from late_interaction_kernels_b200.token_layers import gated_feed_forward

    wt = wdt or dt
    t = {"x": rand(m, k, dt=dt), "wg": rand(f, k, dt=wt, scale=1.5 * k**-0.5), "wu": rand(f, k, dt=wt, scale=k**-0.5), "wd": rand(o, f, dt=wt, scale=f**-0.5)}
    if bias:
        t |= {"bg": rand(f, dt=wt), "bu": rand(f, dt=wt), "bd": rand(o, dt=wt)}
    if residual:
        t["r"] = rand(m, o, dt=dt)
    for v in t.values():
        v.requires_grad_()
    args = [t["x"], t["wg"], t["wu"], t["wd"], t.get("bg"), t.get("bu"), t.get("bd")]
    y = gated_feed_forward(*args, activation=act, residual=t.get("r"))
    assert y.shape == (m, o) and y.dtype == dt
    dy = rand(m, o, dt=dt)
    got = dict(zip(t, torch.autograd.grad(y, list(t.values()), dy)))
    for s in t:
        assert got[s].dtype == t[s].dtype and got[s].shape == t[s].shape
    v = {s: c.detach().to(dt).double() for s, c in t.items()}
    u = unit(dt)
    z, z_err = product(v["x"], v["wg"])
    p, p_err = product(v["x"], v["wu"])
    if bias:
        z, p = z + v["bg"], p + v["bu"]
        z_err, p_err = z_err + E * z.abs(), p_err + E * p.abs()
    a, a_err = act64(z, act), SLOPE * z_err + (act_err(z, dt) if act else 0)
    h = a * p
    h_err = a_err * (p.abs() + p_err) + a.abs() * p_err + E * h.abs()
    h_err = h_err + u * (h.abs() + h_err) + floor(dt)
    y64, y_err = product(h, v["wd"])
    y_err = y_err + mm(h_err, v["wd"].abs().t())
    if bias:
        y64, y_err = y64 + v["bd"], y_err + E * (y64 + v["bd"]).abs()
    if residual:
        y64 = y64 + v["r"]
        y_err = y_err + E * y64.abs()
    near(y.detach(), y64, y_err, "y")
    d = dy.double()
    dh, dh_err = product(d, v["wd"].t())
    s = slope64(z, act)
    s_err = CURVE * z_err + act_err(z, dt) if act and act != "relu" else torch.zeros_like(z)
    if act == "relu":
        s_err = torch.where(z.abs() <= z_err, torch.ones_like(z), s_err)
    dg, du = dh * p * s, dh * a
    fg, fu = (p * s).abs(), a.abs()  # the factors that are kept
    fg_err = p_err * (s.abs() + s_err) + p.abs() * s_err + E * fg
    fg_err, fu_err = fg_err + u * (fg + fg_err) + floor(dt), a_err + u * (fu + a_err) + floor(dt)
    dg_err = dh_err * (fg + fg_err) + dh.abs() * fg_err + E * dg.abs()
    du_err = dh_err * (fu + fu_err) + dh.abs() * fu_err + E * du.abs()
    dg_err = dg_err + u * (dg.abs() + dg_err) + floor(dt)
    du_err = du_err + u * (du.abs() + du_err) + floor(dt)
    dx1, e1 = product(dg, v["wg"].t())
    dx2, e2 = product(du, v["wu"].t())
    near(got["x"], dx1 + dx2, 2 * (e1 + e2) + mm(dg_err, v["wg"].abs()) + mm(du_err, v["wu"].abs()), "dx")
    for name, g, err in (("wg", dg, dg_err), ("wu", du, du_err)):
        w64, e = product(g.t(), v["x"].t())
        near(got[name], w64, e + mm(err.t(), v["x"].abs()), name)
    w64, e = product(d.t(), h.t())
    near(got["wd"], w64, e + mm(d.abs().t(), h_err), "wd")
    if bias:
        for name, g, err in (("bg", dg, dg_err), ("bu", du, du_err), ("bd", d, torch.zeros_like(d))):
            near(got[name], g.sum(0), err.sum(0) + 2 * m * E * g.abs().sum(0), name)
    if residual:
        assert torch.equal(got["r"], dy)
    with torch.no_grad():
        assert torch.equal(gated_feed_forward(*args, activation=act, residual=t.get("r")), y)


GATED = [(1, 1, 1, 1), (1, 16, 40, 8), (3, 5, 7, 9), (8, 768, 512, 768), (16, 64, 2048, 64), (17, 384, 1100, 384), (40, 128, 96, 136), (128, 256, 128, 256), (130, 264, 200, 72),
         (257, 65, 129, 33), (600, 768, 512, 768), (2050, 128, 320, 128), (9000, 64, 40, 64),
         (1500, 300, 700, 260), (3001, 257, 515, 129), (50, 1, 3, 2), (260, 2600, 300, 40), (400, 40, 2800, 136), (5200, 136, 264, 392)]


@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("i", range(len(GATED)))
def test_gated_shapes(dt, i):
    gated_case(*GATED[i], dt, ACTS[1 + (i + 1) % 6], i % 2 == 1, i % 3 != 1)


@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("act", ACTS)
def test_gated_activations(dt, act):
    gated_case(150, 192, 264, 192, dt, act, True, True)


def test_gated_fp32_parameters():
    gated_case(70, 128, 192, 128, BF16, "silu", True, True, wdt=FP32)


# ----------------------------------------------------------------------------- what a program puts around the calls
def head(x, p):
    from late_interaction_kernels_b200.token_layers import gated_feed_forward, layer_norm, linear

    h = layer_norm(x, p["ln_w"], p["ln_b"])
    h = gated_feed_forward(h, p["wg"], p["wu"], p["wd"], activation="gelu", residual=h)
    return linear(h, p["w"], p["b"], activation="gelu_tanh", residual=h)


def head_params(k, f, dt):
    p = {"ln_w": rand(k, dt=dt, scale=0.1, shift=1.0), "ln_b": rand(k, dt=dt, scale=0.1), "wg": rand(f, k, dt=dt, scale=k**-0.5), "wu": rand(f, k, dt=dt, scale=k**-0.5),
         "wd": rand(k, f, dt=dt, scale=f**-0.5), "w": rand(k, k, dt=dt, scale=k**-0.5), "b": rand(k, dt=dt, scale=0.1)}
    return {n: t.requires_grad_() for n, t in p.items()}


def head64(x, p):
    h = torch.nn.functional.layer_norm(x, x.shape[-1:], p["ln_w"], p["ln_b"])
    h = mm(act64(mm(h, p["wg"].t()), "gelu") * mm(h, p["wu"].t()), p["wd"].t()) + h
    return act64(mm(h, p["w"].t()) + p["b"], "gelu_tanh") + h


@pytest.mark.parametrize("dt", [BF16, FP32])
def test_a_token_head_in_front_of_the_scores(dt):
    """hidden states -> layer norm -> gated block -> projection layer -> document head -> scores, and every gradient."""
    from late_interaction_kernels_b200.fused_head import maxsim_from_hidden
    from oracle import maxsim_oracle as O

    Nd, Ld, k = 6, 90, 256
    hidden = rand(Nd, Ld, k, dt=dt).requires_grad_()
    Q = torch.nn.functional.normalize(rand(2, 16, 128, dt=FP32), dim=-1).to(dt)
    W = rand(128, k, dt=dt, scale=k**-0.5).requires_grad_()
    p = head_params(k, 512, dt)
    tokens = head(hidden, p)
    assert tokens.shape == hidden.shape
    scores = maxsim_from_hidden(Q, tokens, W)
    # the layers' roundings: seven in a row, each at most u of values of the same size, so 7 u sqrt(..) stays below 16 u in the 2-norm
    p64 = {n: t.detach().double().requires_grad_() for n, t in p.items()}
    h64 = hidden.detach().double().requires_grad_()
    t64 = head64(h64, p64)
    rel = lambda a, b: float((a.detach().double() - b.detach()).norm() / b.detach().norm())
    assert rel(tokens, t64) < 16 * unit(dt) + 1e-6
    want = O.maxsim_from_hidden(*(t.detach().float().cpu().numpy() for t in (Q, tokens, W)), None, None)
    assert O.rel_err(scores.detach().float().cpu().numpy(), want) < 2e-2
    # gradients of the layers for a given gradient of the tokens: as many roundings again on the way back
    d = rand(Nd, Ld, k, dt=dt)
    leaves = [hidden, *p.values()]
    got = torch.autograd.grad(tokens, leaves, d, retain_graph=True)
    ref = torch.autograd.grad(t64, [h64, *p64.values()], d.double())
    for g, r in zip(got, ref):
        assert rel(g, r) < 32 * unit(dt) + 4e-6
    scores.sum().backward()
    for t in (hidden, W, *p.values()):
        assert t.grad is not None and torch.isfinite(t.grad).all() and t.grad.abs().max() > 0


def test_gradients_against_differences():
    """fp32, central differences of the 64-bit scalar: the slopes that training follows."""
    from late_interaction_kernels_b200.token_layers import gated_feed_forward, layer_norm, linear

    torch.manual_seed(3)
    k = 24
    p = head_params(k, 40, FP32)
    x = rand(11, k, dt=FP32).requires_grad_()
    d = rand(11, k, dt=FP32)
    got = torch.autograd.grad(head(x, p), [x, *p.values()], d)
    leaves = {"x": x, **p}
    for (name, t), g in zip(leaves.items(), got):
        v = {n: c.detach().double() for n, c in leaves.items()}
        dirn = torch.randn_like(v[name])
        step = 1e-5

        def loss(s):
            w = dict(v)
            w[name] = v[name] + s * dirn
            return float((head64(w.pop("x"), w) * d.double()).sum())

        slope = (loss(step) - loss(-step)) / (2 * step)
        # differences: third derivative times step^2, 1e-10 here; the kernels: fp32 through seven layers, sums of 264 terms
        scale = float(g.double().norm() * dirn.norm())
        assert abs(float((g.double() * dirn).sum()) - slope) < 1e-5 * scale, name


@pytest.mark.parametrize("dt", [BF16, FP32])
def test_gradients_are_deterministic_and_only_where_asked(dt):
    p = head_params(128, 256, dt)
    x = rand(3000, 128, dt=dt).requires_grad_()
    d = rand(3000, 128, dt=dt)
    leaves = [x, *p.values()]
    a = torch.autograd.grad(head(x, p), leaves, d)
    b = torch.autograd.grad(head(x, p), leaves, d)
    for s, t in zip(a, b):
        assert torch.equal(s, t)
    for i, t in enumerate(leaves):
        for c in leaves:
            c.requires_grad_(c is t)
        (only,) = torch.autograd.grad(head(x, p), [t], d)
        assert torch.equal(only, a[i])
    for c in leaves:
        c.requires_grad_(True)


def test_steps_on_two_streams_side_by_side():
    p = head_params(256, 512, BF16)
    data = [(rand(700, 256, dt=BF16).requires_grad_(), rand(700, 256, dt=BF16)) for _ in range(2)]

    def step(x, d):
        y = head(x, p)
        return [y.detach(), *torch.autograd.grad(y, [x, *p.values()], d)]

    want = [step(*d) for d in data]
    streams = [torch.cuda.Stream() for _ in data]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(*data[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            for a, b in zip(g, want[i]):
                assert torch.equal(a, b)


def test_steps_from_two_threads():
    from concurrent.futures import ThreadPoolExecutor

    p = head_params(160, 320, BF16)
    data = [(rand(n, 160, dt=BF16).requires_grad_(), rand(n, 160, dt=BF16)) for n in (5, 900)]

    def steps(i):
        x, d = data[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            out = []
            for _ in range(10):
                y = head(x, p)
                out.append([y.detach(), *torch.autograd.grad(y, [x, *p.values()], d)])
            torch.cuda.current_stream().synchronize()
        return out

    torch.cuda.synchronize()
    want = [steps(i)[0] for i in range(2)]
    with ThreadPoolExecutor(2) as pool:
        got = list(pool.map(steps, range(2)))
    for i in range(2):
        for g in got[i]:
            for a, b in zip(g, want[i]):
                assert torch.equal(a, b)


def test_what_is_kept_may_wait_on_the_host():
    p = head_params(96, 160, BF16)
    x, d = rand(70, 96, dt=BF16).requires_grad_(), rand(70, 96, dt=BF16)
    leaves = [x, *p.values()]
    want = torch.autograd.grad(head(x, p), leaves, d)
    with torch.autograd.graph.save_on_cpu():
        y = head(x, p)
    for a, b in zip(torch.autograd.grad(y, leaves, d), want):
        assert torch.equal(a, b)
    with torch.inference_mode():
        assert torch.equal(head(x, p), y)


def test_a_backward_pass_may_run_twice():
    p = head_params(96, 160, FP32)
    x, d = rand(333, 96, dt=FP32).requires_grad_(), rand(333, 96, dt=FP32)
    y = head(x, p)
    leaves = [x, *p.values()]
    a = torch.autograd.grad(y, leaves, d, retain_graph=True)
    b = torch.autograd.grad(y, leaves, d)
    for s, t in zip(a, b):
        assert torch.equal(s, t)
    with pytest.raises(RuntimeError):  # what it kept is gone
        torch.autograd.grad(y, leaves, d)


def test_offsets_beyond_32_bits():
    """Results of more than 2^31 elements: the last rows are those of a call of their own."""
    from late_interaction_kernels_b200.token_layers import gated_feed_forward, layer_norm, linear

    if torch.cuda.mem_get_info()[0] < 40e9:
        pytest.skip("needs 40 GB")
    m = 530000
    with torch.no_grad():
        x, w, b = rand(m, 16, dt=BF16), rand(4096, 16, dt=BF16), rand(4096, dt=BF16)
        y = linear(x, w, b, activation="silu")
        assert y.numel() > 2**31
        tail = linear(x[-5000:], w, b, activation="silu")
        assert torch.equal(y[-5000:], tail)
        n = layer_norm(y)
        assert torch.equal(n[-5000:], layer_norm(tail))
        del n
        back = linear(y, rand(24, 4096, dt=BF16).fill_(2**-6))
        near(back[-64:], *(lambda v, e: (v, e))(*product(tail[-64:].double(), torch.full((24, 4096), 2.0**-6, dtype=torch.float64, device="cuda"))), "back")
        del y, back
    x.requires_grad_()
    wg = rand(4096, 16, dt=BF16)
    y = gated_feed_forward(x, wg, w, w.t())
    (dx,) = torch.autograd.grad(y, [x], torch.ones_like(y))
    few = x.detach()[-5000:].clone().requires_grad_()
    z = gated_feed_forward(few, wg, w, w.t())
    # (5000 rows have their sums over 4096 cut into shares: fp32 sums in another order, each element rounded once, so at most a step of 2 u apart)
    for a, b in ((y[-5000:], z), (dx[-5000:], torch.autograd.grad(z, [few], torch.ones_like(z))[0])):
        assert float((a.double() - b.double()).norm() / b.double().norm()) < 2 * unit(BF16)


def test_a_step_in_a_cuda_graph_and_on_another_stream():
    from late_interaction_kernels_b200 import check_device_status

    p = head_params(256, 512, BF16)
    x, d = rand(700, 256, dt=BF16).requires_grad_(), rand(700, 256, dt=BF16)
    leaves = [x, *p.values()]

    def step():
        y = head(x, p)
        return [y.detach(), *torch.autograd.grad(y, leaves, d)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    want = step()
    for a, b in zip(on_side, want):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):  # two graphs side by side, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for seed in range(3):
        torch.manual_seed(seed)
        with torch.no_grad():
            x.copy_(rand(700, 256, dt=BF16))
            d.copy_(rand(700, 256, dt=BF16))
        for g, _ in graphs:
            g.replay()
        eager = step()
        for _, out in graphs:
            for a, b in zip(out, eager):
                assert torch.equal(a, b)
    check_device_status()


def test_capture_beside_a_live_eager_graph_is_refused():
    from late_interaction_kernels_b200.token_layers import linear

    x, w = rand(8, 64, dt=BF16), rand(32, 64, dt=BF16).requires_grad_()
    alive = linear(x, w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        keep = x * 1
        with pytest.raises(RuntimeError, match="still alive"):
            linear(x, w)
    torch.cuda.synchronize()
    del alive
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        (grad,) = torch.autograd.grad(linear(x, w), [w], torch.ones(8, 32, device="cuda", dtype=BF16))
    g.replay()
    assert torch.equal(grad, torch.autograd.grad(linear(x, w), [w], torch.ones(8, 32, device="cuda", dtype=BF16))[0])
    del keep


def test_second_derivatives_and_tangents_are_refused():
    from late_interaction_kernels_b200.token_layers import gated_feed_forward, layer_norm, linear

    x, w = rand(8, 64, dt=FP32).requires_grad_(), rand(64, 64, dt=FP32).requires_grad_()
    for fn in (lambda: layer_norm(x), lambda: linear(x, w), lambda: gated_feed_forward(x, w, w, w)):
        (g,) = torch.autograd.grad(fn().square().sum(), [x], create_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            g.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        t = torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x))
        for fn in (lambda: layer_norm(t), lambda: linear(t, w.detach()), lambda: gated_feed_forward(t, w, w, w)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                fn()


def test_checkpointing_shared_weights_and_saved_values_changed_in_place():
    from torch.utils.checkpoint import checkpoint

    from late_interaction_kernels_b200.token_layers import gated_feed_forward, linear

    p = head_params(128, 192, BF16)
    x, d = rand(2, 50, 128, dt=BF16).requires_grad_(), rand(2, 50, 128, dt=BF16)
    leaves = [x, *p.values()]
    a = torch.autograd.grad(head(x, p), leaves, d)
    b = torch.autograd.grad(checkpoint(lambda t: head(t, p), x, use_reentrant=False), leaves, d)
    for s, t in zip(a, b):
        assert torch.equal(s, t)
    # one weight for both projections: its gradient is the sum of the two
    w = rand(192, 128, dt=FP32).requires_grad_()
    wd = rand(128, 192, dt=FP32)
    xs, ds = rand(30, 128, dt=FP32), rand(30, 128, dt=FP32)
    (both,) = torch.autograd.grad(gated_feed_forward(xs, w, w, wd), [w], ds)
    w2 = w.detach().clone().requires_grad_()
    g1, g2 = torch.autograd.grad(gated_feed_forward(xs, w, w2, wd), [w, w2], ds)
    assert torch.equal(both, g1 + g2)
    y = linear(x, p["w"], activation="gelu")
    with torch.no_grad():
        p["w"].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, [x], torch.ones_like(y))


def test_empty_batches():
    p = head_params(64, 96, BF16)
    x = rand(0, 5, 64, dt=BF16).requires_grad_()
    y = head(x, p)
    assert y.shape == (0, 5, 64)
    y.sum().backward()
    assert x.grad.shape == x.shape
    for t in p.values():
        assert t.grad is not None and not t.grad.any()



# ----------------------------------------------------------------------------- refusals
def test_refusals():
    from late_interaction_kernels_b200.token_layers import gated_feed_forward, layer_norm, linear

    x, w, b = rand(4, 8, dt=BF16), rand(6, 8, dt=BF16), rand(6, dt=BF16)
    wd = rand(8, 6, dt=BF16)
    one = rand(1, 1, dt=BF16)
    bad = [
        (lambda: layer_norm(x, b), r"weight must be \[8\]"), (lambda: layer_norm(x, None, b), r"bias must be \[8\]"), (lambda: layer_norm(x, eps=-1.0), "eps"),
        (lambda: layer_norm(x, eps=float("nan")), "eps"), (lambda: layer_norm(x.to(torch.float64)), "not supported"), (lambda: layer_norm(x[:, :0]), "at least one feature"),
        (lambda: layer_norm(x, rand(8, dt=BF16).cpu()), "same device"), (lambda: layer_norm(x[0, 0]), "at least one dimension"),
        (lambda: linear(x, w[:, :7]), r"weight must be"), (lambda: linear(x, b), "weight must be"), (lambda: linear(x, w[:0]), "weight must be"),
        (lambda: linear(x, w, b[:5]), r"bias must be \[6\]"), (lambda: linear(x, w, activation="swish"), "activation must be"),
        (lambda: linear(x, w, residual=rand(6, dt=BF16)), "residual must have"), (lambda: linear(x, w, residual=rand(1, 6, dt=BF16)), "residual must have"),
        (lambda: linear(x, w.to(torch.int32)), "not supported"), (lambda: linear(x, w, b.cpu()), "same device"), (lambda: linear(x[:, :0], w[:, :0]), "at least one feature"),
        (lambda: gated_feed_forward(x, w, w[:5], wd), "w_up must be"), (lambda: gated_feed_forward(x, w, w, wd[:, :5]), "w_down must be"),
        (lambda: gated_feed_forward(x, w, w, wd, b_down=b), r"b_down must be \[8\]"), (lambda: gated_feed_forward(x, w, w, wd, residual=x[:3]), "residual must have"),
        (lambda: gated_feed_forward(x, w, w, wd, activation="x"), "activation must be"),
        # sizes beyond what the kernels count with
        (lambda: linear(one.expand(1, 2**32 + 8), one.expand(1, 2**32 + 8)), "less than 2"), (lambda: linear(one, one.expand(2**32 + 8, 1)), "less than 2"),
        (lambda: gated_feed_forward(one, one.expand(2**32, 1), one.expand(2**32, 1), one.expand(1, 2**32)), "less than 2"),
        (lambda: gated_feed_forward(one, one, one, one.expand(2**32, 1)), "less than 2"),
    ]
    for fn, text in bad:
        with pytest.raises(ValueError, match=text):
            fn()
