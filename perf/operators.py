"""The layers that stand between an encoder's hidden states and the document head, as cases that can be timed and compared.

  layer_norm           layer norm over the last dimension, and its backward pass
  linear               ``act(x @ W.T + b) + residual``, and its backward pass
  gated_feed_forward   ``(act(x @ Wg.T + bg) * (x @ Wu.T + bu)) @ Wd.T + bd + residual``, and its backward pass

With ``own`` false the operators are computed from elementary torch operations in 32 bits and rounded once at the end;
with ``own`` true the same inputs go to this package's entry points.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ITEM = {"bf16": 2, "fp16": 2, "fp32": 4}
ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh", "tanh", "sigmoid")


def listed():
    return [
        # one query's 32 tokens on their way to the scorer: nothing but latency
        {"name": "norm_query", "op": "layer_norm", "tokens": 32, "width": 768, "dtype": "bf16", "affine": True, "train": False},
        # the documents of a training batch (256 of 256 tokens), forward and backward: bandwidth
        {"name": "norm_train", "op": "layer_norm", "tokens": 65536, "width": 768, "dtype": "bf16", "affine": True, "train": True},
        # fp32 training on packed documents, an odd width: rows that no vector load can assume aligned
        {"name": "norm_odd_fp32", "op": "layer_norm", "tokens": 9001, "width": 1023, "dtype": "fp32", "affine": True, "train": True},
        # a single token through a projection layer while a stream of text is encoded
        {"name": "linear_token", "op": "linear", "tokens": 1, "k": 768, "n": 768, "dtype": "bf16", "act": "gelu", "bias": True, "residual": True, "train": False},
        # a few queries of 32 tokens down to the scored width
        {"name": "linear_queries", "op": "linear", "tokens": 128, "k": 768, "n": 128, "dtype": "fp16", "act": "none", "bias": False, "residual": False, "train": False},
        # a training step's documents through a residual projection layer
        {"name": "linear_train", "op": "linear", "tokens": 65536, "k": 768, "n": 768, "dtype": "bf16", "act": "gelu", "bias": True, "residual": True, "train": True},
        # sizes that no tile divides and rows that are not 16-byte aligned
        {"name": "linear_odd", "op": "linear", "tokens": 7681, "k": 1001, "n": 333, "dtype": "fp16", "act": "relu", "bias": True, "residual": True, "train": True},
        # a head trained in fp32
        {"name": "linear_fp32", "op": "linear", "tokens": 8192, "k": 768, "n": 512, "dtype": "fp32", "act": "tanh", "bias": True, "residual": False, "train": True},
        # a single token through a gated block: the weights' bytes and two launches
        {"name": "gated_token", "op": "gated", "tokens": 1, "k": 768, "f": 2048, "dtype": "bf16", "act": "silu", "bias": False, "residual": True, "train": False},
        # sixteen queries encoded together
        {"name": "gated_queries", "op": "gated", "tokens": 512, "k": 768, "f": 2048, "dtype": "bf16", "act": "gelu", "bias": False, "residual": True, "train": False},
        # ragged fp16 training step with biases
        {"name": "gated_odd", "op": "gated", "tokens": 5003, "k": 384, "f": 1100, "dtype": "fp16", "act": "gelu_tanh", "bias": True, "residual": False, "train": True},
        # the documents of a training batch through a wide block, forward and backward: the largest
        {"name": "gated_train", "op": "gated", "tokens": 65536, "k": 1024, "f": 4096, "dtype": "bf16", "act": "silu", "bias": False, "residual": True, "train": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A feature count: mostly of whole vectors, as models have them, and odd ones among them."""
    step = rng.choice((64, 64, 8, 8, 1))
    return max(lo, _log(rng, lo, hi) // step * step)


def draw(rng):
    op = rng.choice(("layer_norm", "linear", "linear", "gated", "gated"))
    case = {"op": op, "tokens": _log(rng, 1, 65536), "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")), "train": rng.random() < 0.6}
    if op == "layer_norm":
        return case | {"width": _width(rng, 16, 4096), "affine": rng.random() < 0.8}
    case |= {"act": rng.choice(ACTIVATIONS), "bias": rng.random() < 0.5, "residual": rng.random() < 0.5}
    if op == "linear":
        return case | {"k": _width(rng, 32, 2048), "n": _width(rng, 16, 2048)}
    case |= {"k": _width(rng, 32, 1024), "f": _width(rng, 32, 4096)}
    if case["dtype"] == "fp32":  # the wide blocks are not run in fp32 on many tokens
        case["tokens"] = min(case["tokens"], 16384)
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, tokens = DTYPES[case["dtype"]], case["tokens"]

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dt)

    k = case["width"] if case["op"] == "layer_norm" else case["k"]
    # hidden states: features of differing spread and mean, as an encoder's have
    spread = torch.exp(0.5 * torch.randn(k, generator=g, device="cuda"))
    centre = 0.3 * torch.randn(k, generator=g, device="cuda")
    x = (torch.randn(tokens, k, generator=g, device="cuda").mul_(spread).add_(centre)).to(dt)
    s = {"case": case, "x": x, "dy": None}
    out = k
    if case["op"] == "layer_norm":
        s |= {"weight": normal(k, scale=0.2, shift=1.0), "bias": normal(k, scale=0.1)} if case["affine"] else {"weight": None, "bias": None}
    elif case["op"] == "linear":
        out = case["n"]
        s |= {"weight": normal(out, k, scale=k**-0.5), "bias": normal(out, scale=0.1) if case["bias"] else None}
        s |= {"residual": normal(tokens, out) if case["residual"] else None}
    else:
        f = case["f"]
        s |= {"w_gate": normal(f, k, scale=k**-0.5), "w_up": normal(f, k, scale=k**-0.5), "w_down": normal(k, f, scale=f**-0.5)}
        s |= {n: normal(m, scale=0.1) if case["bias"] else None for n, m in (("b_gate", f), ("b_up", f), ("b_down", k))}
        s |= {"residual": normal(tokens, k) if case["residual"] else None}
    if case["train"]:
        s["dy"] = normal(tokens, out)
        for n, t in s.items():
            if n not in ("case", "dy") and t is not None:
                t.requires_grad_(True)
    return s


def _names(state):
    return [n for n, t in state.items() if n not in ("case", "dy") and t is not None]


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"layer_norm": _plain_norm, "linear": _plain_linear, "gated": _plain_gated}[state["case"]["op"]](state)


def _run_own(s):
    from late_interaction_kernels_b200.token_layers import gated_feed_forward, layer_norm, linear

    case = s["case"]
    act = None if case.get("act") in (None, "none") else case["act"]
    if case["op"] == "layer_norm":
        y = layer_norm(s["x"], s["weight"], s["bias"], eps=1e-5)
    elif case["op"] == "linear":
        y = linear(s["x"], s["weight"], s["bias"], activation=act, residual=s["residual"])
    else:
        y = gated_feed_forward(s["x"], s["w_gate"], s["w_up"], s["w_down"], b_gate=s["b_gate"], b_up=s["b_up"], b_down=s["b_down"], activation=act, residual=s["residual"])
    if not case["train"]:
        return {"y": y}
    names = _names(s)
    return {"y": y.detach()} | {"d_" + n: t for n, t in zip(names, torch.autograd.grad(y, [s[n] for n in names], s["dy"]))}


# ---- the plain forms: elementary operations in fp32, gradients from their formulas ----


def _f(t):
    return None if t is None else t.float()


def _act(z, act):
    if act == "none":
        return z
    if act == "relu":
        return z.clamp(min=0)
    if act == "sigmoid":
        return torch.sigmoid(z)
    if act == "tanh":
        return torch.tanh(z)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))


def _act_slope(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "sigmoid":
        s = torch.sigmoid(z)
        return s * (1 - s)
    if act == "tanh":
        return 1 - torch.tanh(z).square()
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def _plain_norm(s):
    x, w, b = _f(s["x"]), _f(s["weight"]), _f(s["bias"])
    dt = s["x"].dtype
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    inv = torch.rsqrt(centred.square().mean(1, keepdim=True) + 1e-5)
    hat = centred * inv
    y = hat if w is None else hat * w + b
    out = {"y": y.to(dt)}
    if s["dy"] is None:
        return out
    dy = _f(s["dy"])
    g = dy if w is None else dy * w
    dx = inv * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
    out |= {"d_x": dx.to(dt)}
    return out if w is None else out | {"d_weight": (dy * hat).sum(0).to(dt), "d_bias": dy.sum(0).to(dt)}


def _plain_linear(s):
    case, dt = s["case"], s["x"].dtype
    x, w = _f(s["x"]), _f(s["weight"])
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + _f(s["bias"])
    y = _act(z, case["act"])
    if s["residual"] is not None:
        y = y + _f(s["residual"])
    out = {"y": y.to(dt)}
    if s["dy"] is None:
        return out
    dz = _f(s["dy"]) * _act_slope(z, case["act"])
    out |= {"d_x": (dz @ w).to(dt), "d_weight": (dz.t() @ x).to(dt)}
    if s["bias"] is not None:
        out["d_bias"] = dz.sum(0).to(dt)
    return out if s["residual"] is None else out | {"d_residual": s["dy"]}


def _plain_gated(s):
    case, dt = s["case"], s["x"].dtype
    x, wg, wu, wd = _f(s["x"]), _f(s["w_gate"]), _f(s["w_up"]), _f(s["w_down"])
    gate, up = x @ wg.t(), x @ wu.t()
    if case["bias"]:
        gate, up = gate + _f(s["b_gate"]), up + _f(s["b_up"])
    a = _act(gate, case["act"])
    h = a * up
    y = h @ wd.t()
    if case["bias"]:
        y = y + _f(s["b_down"])
    if s["residual"] is not None:
        y = y + _f(s["residual"])
    out = {"y": y.to(dt)}
    if s["dy"] is None:
        return out
    dy = _f(s["dy"])
    dh = dy @ wd
    d_gate, d_up = dh * up * _act_slope(gate, case["act"]), dh * a
    out |= {"d_x": (d_gate @ wg + d_up @ wu).to(dt), "d_w_gate": (d_gate.t() @ x).to(dt), "d_w_up": (d_up.t() @ x).to(dt), "d_w_down": (dy.t() @ h).to(dt)}
    if case["bias"]:
        out |= {"d_b_gate": d_gate.sum(0).to(dt), "d_b_up": d_up.sum(0).to(dt), "d_b_down": dy.sum(0).to(dt)}
    return out if s["residual"] is None else out | {"d_residual": s["dy"]}


# ---- what a pass cannot do without ----


def work(case):
    b, m = ITEM[case["dtype"]], case["tokens"]
    train = case["train"]
    if case["op"] == "layer_norm":
        w = case["width"]
        params = 2 * w if case["affine"] else 0
        return {"bytes": b * ((4 if train else 2) * m * w + (2 if train else 1) * params), "flops": (19 if train else 8) * m * w}
    k = case["k"]
    if case["op"] == "linear":
        n = case["n"]
        params, flops, out = n * k + (n if case["bias"] else 0), 2 * m * n * k, n
    else:
        f = case["f"]
        params, flops, out = 3 * f * k + (2 * f + k if case["bias"] else 0), 6 * m * f * k, k
    rows = m * k + m * out * (2 if case["residual"] else 1)  # x, residual; y
    if train:  # dy; dx and a residual's gradient; the parameters' gradients
        rows += m * out + m * k + (m * out if case["residual"] else 0)
        params, flops = 2 * params, 3 * flops
    return {"bytes": b * (rows + params), "flops": flops}


# ---- the definition in 64 bits: every function written once, derivatives by automatic differentiation ----


def exact(case, seed):
    state = prepare(case, seed)
    names = _names(state)
    v = {n: state[n].detach().double().requires_grad_(case["train"]) for n in names}
    x = v["x"]
    with torch.set_grad_enabled(case["train"]):
        if case["op"] == "layer_norm":
            var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
            y = (x - mean) / (var + 1e-5).sqrt()
            if case["affine"]:
                y = torch.addcmul(v["bias"], y, v["weight"])
        elif case["op"] == "linear":
            y = _exact_act(_affine(x, v["weight"], v.get("bias")), case["act"])
        else:
            h = _exact_act(_affine(x, v["w_gate"], v.get("b_gate")), case["act"]) * _affine(x, v["w_up"], v.get("b_up"))
            y = _affine(h, v["w_down"], v.get("b_down"))
        if "residual" in v:
            y = y + v["residual"]
    if not case["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, [v[n] for n in names], state["dy"].double())
    return {"y": y.detach()} | {"d_" + n: t for n, t in zip(names, grads)}


def _affine(x, w, b):
    y = torch.einsum("mk,nk->mn", x, w)
    return y if b is None else y + b[None, :]


def _exact_act(z, act):
    phi = {"none": None, "relu": lambda t: (t > 0).double(), "silu": lambda t: 1 / (1 + torch.exp(-t)), "gelu": torch.special.ndtr,
           "gelu_tanh": lambda t: 1 / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (t + 0.044715 * t**3)))}
    if act == "tanh":
        return 2 / (1 + torch.exp(-2 * z)) - 1
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    return z if act == "none" else z * phi[act](z)
