"""What is measured of the feed-forward operators: layer norm, the linear
layer with its epilogue, and the products grouped by expert, each forwards
and backwards.

`run` computes a case either in plain float32 torch operations (`own` false)
or with this package's kernels (`own` true) on the same inputs.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
ELEMENT_BYTES = {"bfloat16": 2, "float16": 2, "float32": 4}
EPS = 1e-5


def _package():
    """This repository's package; its folder's name is no Python identifier."""
    folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                          "php-gpu-tensors_b200")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import phptensors
    return phptensors


# ------------------------------------------------------------------ cases
def _norm(name, direction, dtype, rows, cols):
    return {"name": name, "op": "layer_norm", "direction": direction, "dtype": dtype,
            "rows": rows, "cols": cols}


def _linear(name, direction, dtype, rows, inner, cols, activation, bias=True, residual=False,
            save_pre=False, column_major=False):
    return {"name": name, "op": "linear", "direction": direction, "dtype": dtype, "rows": rows,
            "inner": inner, "cols": cols, "activation": activation, "bias": bias,
            "residual": residual, "save_pre": save_pre, "column_major": column_major}


def _experts(name, direction, dtype, rows, inner, cols, experts, empty, activation, bias=True,
             residual=False, save_pre=False, column_major=False):
    return {"name": name, "op": "experts", "direction": direction, "dtype": dtype, "rows": rows,
            "inner": inner, "cols": cols, "experts": experts, "empty": empty,
            "activation": activation, "bias": bias, "residual": residual, "save_pre": save_pre,
            "column_major": column_major}


def listed():
    return [
        # serving: the norm in front of a layer for eight sequences, one new
        # token each; the time is launch latency
        _norm("norm_decode_bf16", "forward", "bfloat16", 8, 4096),
        # a float32 model with widths that are a multiple of nothing: rows
        # start at every alignment
        _norm("norm_forward_f32_odd", "forward", "float32", 3001, 1531),
        # training in float16 on a ragged batch, rows that are only 4-byte aligned
        _norm("norm_backward_f16_odd", "backward", "float16", 2777, 2050),
        # training: the gradient of a wide layer's norm over a full batch of tokens
        _norm("norm_backward_bf16_large", "backward", "bfloat16", 16384, 4096),
        # serving: one new token for each of eight sequences through a square
        # projection back into the residual stream; the weight's bytes bound it
        _linear("linear_decode_bf16", "forward", "bfloat16", 8, 4096, 4096, "none",
                residual=True),
        # a prompt through a layer whose sizes are odd in every direction
        _linear("linear_prompt_f16_odd", "forward", "float16", 1999, 1021, 2055, "gelu"),
        # the square layer of this repository's float32 MLP set (batch 4096)
        _linear("linear_f32", "forward", "float32", 4096, 1024, 1024, "tanh", residual=True),
        # training: the widening layer with its activation; the pre-activation
        # is kept for the backward pass
        _linear("linear_train_bf16", "forward", "bfloat16", 16384, 2048, 8192, "gelu_tanh",
                save_pre=True),
        # its backward pass: gradients of the activation, input, weight and bias
        _linear("linear_backward_bf16", "backward", "bfloat16", 8192, 2048, 8192, "gelu_tanh"),
        # serving: sixteen tokens, two experts each, out of 32 experts
        _experts("experts_decode_bf16", "forward", "bfloat16", 32, 2048, 1024, 32, 0, "silu",
                 bias=False),
        # a prompt over 64 experts, some of which get nothing
        _experts("experts_prompt_bf16", "forward", "bfloat16", 8192, 2048, 1408, 64, 5, "silu",
                 save_pre=True),
        # training: the backward pass of a batch over 16 experts
        _experts("experts_backward_f16", "backward", "float16", 16384, 2048, 2048, 16, 1,
                 "gelu"),
    ]


MOST_FLOPS = 5.4e11          # the largest listed case (linear_backward_bf16: 5.5e11)


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """Half of the widths are multiples of 64, a quarter of 8, the rest any."""
    n = _between(rng, low, high)
    kind = rng.random()
    step = 64 if kind < 0.5 else 8 if kind < 0.75 else 1
    return max(step, n // step * step)


def draw(rng):
    op = rng.choice(["layer_norm", "linear", "experts"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    direction = rng.choice(["forward", "backward"])
    if op == "layer_norm":
        while True:
            c = _norm("", direction, dtype, _between(rng, 1, 32768), _width(rng, 64, 8192))
            if c["rows"] * c["cols"] <= 16384 * 4096 * 2 // ELEMENT_BYTES[dtype]:
                break
    else:
        activation = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu", "tanh", "sigmoid"])
        bias, column_major = rng.random() < 0.7, rng.random() < 0.3
        residual = direction == "forward" and rng.random() < 0.4
        save_pre = direction == "forward" and rng.random() < 0.3
        while True:
            if op == "linear":
                c = _linear("", direction, dtype, _between(rng, 1, 16384), _width(rng, 64, 8192),
                            _width(rng, 64, 8192), activation, bias, residual, save_pre,
                            column_major)
            else:
                experts = rng.choice([4, 8, 16, 32, 60, 64, 128])
                c = _experts("", direction, dtype, _between(rng, 1, 16384),
                             _width(rng, 64, 4096), _width(rng, 64, 4096), experts,
                             rng.choice([0, 0, 1, experts // 4]), activation, bias, residual,
                             save_pre, column_major)
            weights = c["inner"] * c["cols"] * c.get("experts", 1)
            if weights <= 64 * 2048 * 2048 and work(c)["flops"] <= MOST_FLOPS:
                break
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs
def _counts(case, seed):
    """Rows of each expert: a router's skewed shares (the fullest expert gets
    about four times the share of the emptiest), `empty` of them with none."""
    rng = random.Random(seed * 1000003 + 17)
    share = [rng.uniform(1.0, 4.0) for _ in range(case["experts"])]
    for e in rng.sample(range(case["experts"]), case["empty"]):
        share[e] = 0.0
    counts = [0] * case["experts"]
    for e in rng.choices(range(case["experts"]), share, k=case["rows"]):
        counts[e] += 1
    return counts


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dtype):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(dtype)

    rows = case["rows"]
    state = {"case": dict(case)}
    if case["op"] == "layer_norm":
        cols = case["cols"]
        # activations of a residual stream: every channel has its own offset
        # and spread, a few are far wider than the rest
        offset = torch.randn(cols, generator=g, device="cuda") * 0.3 + 0.2
        spread = torch.rand(cols, generator=g, device="cuda") + 0.5
        spread[:: max(1, cols // 4)] *= 8
        x = (torch.randn(rows, cols, generator=g, device="cuda") * spread + offset).to(dtype)
        state["x"] = x
        state["gamma"] = (torch.randn(cols, generator=g, device="cuda") * 0.2 + 1).to(dtype)
        state["beta"] = normal(cols, scale=0.2)
        if case["direction"] == "backward":
            xf = x.float()
            mean = xf.mean(1)
            state["mean"] = mean
            state["rstd"] = ((xf - mean[:, None]).square().mean(1) + EPS).rsqrt()
            state["grad"] = normal(rows, cols)
        return state
    inner, cols = case["inner"], case["cols"]
    lead = [case["experts"]] if case["op"] == "experts" else []
    state["x"] = normal(rows, inner)
    if case["column_major"]:
        w = normal(*lead, cols, inner, scale=inner ** -0.5)
        state["weight"] = w.transpose(-1, -2)
    else:
        state["weight"] = normal(*lead, inner, cols, scale=inner ** -0.5)
    state["bias"] = normal(*lead, cols, scale=0.3) if case["bias"] else None
    state["residual"] = normal(rows, cols) if case["residual"] else None
    if case["direction"] == "backward":
        state["grad"] = normal(rows, cols)
        state["pre"] = normal(rows, cols) if case["activation"] != "none" else None
    if lead:
        counts = _counts(case, seed)
        state["capacity"] = max(counts)
        state["ends"] = torch.tensor(counts).cumsum(0).to(torch.int32).cuda()
    return state


# ------------------------------------------------------------------ plain form
def _activate(z, activation):
    if activation == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if activation == "tanh":
        return torch.tanh(z)
    if activation == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    if activation == "silu":
        return z / (1 + torch.exp(-z))
    if activation == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if activation == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _slope(z, activation):
    if activation == "relu":
        return (z > 0).float()
    if activation == "tanh":
        return 1 - torch.tanh(z).square()
    if activation == "sigmoid":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 - s)
    if activation == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if activation == "gelu":
        return (0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
                + z * torch.exp(-0.5 * z * z) * math.sqrt(0.5 / math.pi))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def _plain_norm(s):
    c, x, gamma = s["case"], s["x"].float(), s["gamma"].float()
    if c["direction"] == "forward":
        mean = x.mean(1)
        centred = x - mean[:, None]
        rstd = (centred.square().mean(1) + EPS).rsqrt()
        y = centred * rstd[:, None] * gamma + s["beta"].float()
        return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}
    grad = s["grad"].float()
    normed = (x - s["mean"][:, None]) * s["rstd"][:, None]
    scaled = grad * gamma
    dx = (scaled - scaled.mean(1, keepdim=True)
          - normed * (scaled * normed).mean(1, keepdim=True)) * s["rstd"][:, None]
    return {"dx": dx.to(s["x"].dtype), "dgamma": (grad * normed).sum(0), "dbeta": grad.sum(0)}


def _plain_finish(s, z):
    c, dtype = s["case"], s["x"].dtype
    y = _activate(z, c["activation"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(dtype)}
    if c["save_pre"]:
        out["pre"] = z.to(dtype)
    return out


def _plain_dz(s):
    grad = s["grad"].float()
    activation = s["case"]["activation"]
    return grad if activation == "none" else grad * _slope(s["pre"].float(), activation)


def _plain_linear(s):
    c, x, w = s["case"], s["x"].float(), s["weight"].float()
    if c["direction"] == "forward":
        z = x @ w
        if s["bias"] is not None:
            z = z + s["bias"].float()
        return _plain_finish(s, z)
    dz = _plain_dz(s)
    out = {"dx": (dz @ w.t()).to(s["x"].dtype), "dw": (x.t() @ dz).to(s["x"].dtype)}
    if c["bias"]:
        out["dbias"] = dz.sum(0)
    return out


def _plain_experts(s):
    """Rows laid out as one padded block per expert, so that one batched
    product serves all of them."""
    c, x, w, ends = s["case"], s["x"].float(), s["weight"].float(), s["ends"].long()
    starts = torch.cat([ends.new_zeros(1), ends[:-1]])
    place = starts[:, None] + torch.arange(s["capacity"], device="cuda")
    filled = (place < ends[:, None])[:, :, None]
    place = place.clamp(max=c["rows"] - 1)
    row = torch.arange(c["rows"], device="cuda")
    expert = torch.searchsorted(ends, row, right=True)
    at = row - starts[expert]

    def spread(t):
        return torch.where(filled, t[place], 0.0)

    if c["direction"] == "forward":
        z = torch.bmm(spread(x), w)[expert, at]
        if s["bias"] is not None:
            z = z + s["bias"].float()[expert]
        return _plain_finish(s, z)
    dz = spread(_plain_dz(s))
    out = {"dx": torch.bmm(dz, w.transpose(1, 2))[expert, at].to(s["x"].dtype),
           "dw": torch.bmm(spread(x).transpose(1, 2), dz).to(s["x"].dtype)}
    if c["bias"]:
        out["dbias"] = dz.sum(1)
    return out


# ------------------------------------------------------------------ the package's calls
def _own(s):
    P, c = _package(), s["case"]

    def arr(name):
        return None if s.get(name) is None else P.CudaArray.from_torch(s[name])

    x = arr("x")
    if c["op"] == "layer_norm":
        if c["direction"] == "forward":
            out = x.layer_norm(arr("gamma"), arr("beta"), EPS, save_stats=True)
            names = ("y", "mean", "rstd")
        else:
            out = P.layer_norm_backward(arr("grad"), x, arr("gamma"), arr("mean"), arr("rstd"))
            names = ("dx", "dgamma", "dbeta")
    elif c["direction"] == "forward":
        options = {"bias": arr("bias"), "activation": c["activation"],
                   "residual": arr("residual"), "save_pre": c["save_pre"]}
        if c["op"] == "linear":
            out = x.linear(arr("weight"), **options)
        else:
            out = x.grouped_linear(arr("weight"), s["ends"], **options)
        out = out if c["save_pre"] else (out,)
        names = ("y", "pre")
    else:
        options = {"pre": arr("pre"), "activation": c["activation"], "bias": c["bias"]}
        if c["op"] == "linear":
            out = P.linear_backward(arr("grad"), x, arr("weight"), **options)
        else:
            out = P.grouped_linear_backward(arr("grad"), x, arr("weight"), s["ends"], **options)
        names = ("dx", "dw", "dbias")
    return {n: t.to_torch() for n, t in zip(names, out) if t is not None}


def run(state):
    if own:
        return _own(state)
    return {"layer_norm": _plain_norm, "linear": _plain_linear,
            "experts": _plain_experts}[state["case"]["op"]](state)


# ------------------------------------------------------------------ what a pass needs
def work(case):
    es, rows = ELEMENT_BYTES[case["dtype"]], case["rows"]
    back = case["direction"] == "backward"
    if case["op"] == "layer_norm":
        n = rows * case["cols"]
        if back:      # x, its gradient and the result's; gamma and two gradients; statistics
            return {"bytes": 3 * n * es + case["cols"] * (es + 8) + rows * 8, "flops": 14 * n}
        return {"bytes": 2 * n * es + case["cols"] * 2 * es + rows * 8, "flops": 8 * n}
    inner, cols, experts = case["inner"], case["cols"], case.get("experts", 1)
    used = experts
    if case["op"] == "experts":       # experts that get a row, on average
        live = experts - case["empty"]
        used = live * (1 - (1 - 1 / live) ** rows)
    weights = used * inner * cols
    active = case["activation"] != "none"
    if back:
        # gradient, pre-activation, input and its gradient; the weight read,
        # its gradient (all experts) written
        size = (rows * (cols * (2 if active else 1) + 2 * inner) + weights
                + experts * inner * cols) * es
        size += experts * cols * 4 if case["bias"] else 0
        flops = 4 * rows * inner * cols
    else:
        size = (rows * (inner + cols * (1 + bool(case["residual"]) + bool(case["save_pre"])))
                + weights + (used * cols if case["bias"] else 0)) * es
        flops = 2 * rows * inner * cols
    return {"bytes": int(size + (4 * experts if case["op"] == "experts" else 0)),
            "flops": int(flops)}


# ------------------------------------------------------------------ in 64 bits
def _f64(t):
    return None if t is None else t.double()


def _exact_activation(z, activation):
    F = torch.nn.functional
    if activation == "none":
        return z
    if activation in ("gelu", "gelu_tanh"):
        return F.gelu(z, approximate="tanh" if activation == "gelu_tanh" else "none")
    return {"relu": F.relu, "silu": F.silu, "tanh": torch.tanh,
            "sigmoid": torch.sigmoid}[activation](z)


def exact(case, seed):
    s = prepare(case, seed)
    x = _f64(s["x"])
    if case["op"] == "layer_norm":
        if case["direction"] == "forward":
            var, mean = torch.var_mean(x, 1, correction=0)
            y = torch.nn.functional.layer_norm(x, x.shape[1:], _f64(s["gamma"]),
                                               _f64(s["beta"]), EPS)
            return {"y": y, "mean": mean, "rstd": (var + EPS) ** -0.5}
        # the chain rule through mean and variance, for the statistics given
        mean, rstd = _f64(s["mean"])[:, None], _f64(s["rstd"])[:, None]
        grad, n = _f64(s["grad"]), x.shape[1]
        dn = grad * _f64(s["gamma"])
        dvar = (dn * (x - mean)).sum(1, keepdim=True) * -0.5 * rstd ** 3
        dmean = -rstd * dn.sum(1, keepdim=True)
        dx = dn * rstd + dvar * 2 * (x - mean) / n + dmean / n
        return {"dx": dx, "dgamma": torch.einsum("rc,rc->c", grad, (x - mean) * rstd),
                "dbeta": torch.einsum("rc->c", grad)}
    w = _f64(s["weight"]).reshape(-1, case["inner"], case["cols"])
    bias = None if s["bias"] is None else _f64(s["bias"]).reshape(-1, case["cols"])
    bounds = [0] + (s["ends"].tolist() if case["op"] == "experts" else [case["rows"]])
    spans = list(zip(bounds[:-1], bounds[1:]))
    if case["direction"] == "forward":
        z = torch.cat([torch.addmm(bias[e], x[a:b], w[e]) if bias is not None else x[a:b] @ w[e]
                       for e, (a, b) in enumerate(spans)])
        y = _exact_activation(z, case["activation"])
        if s["residual"] is not None:
            y = y + _f64(s["residual"])
        return {"y": y, "pre": z} if case["save_pre"] else {"y": y}
    dz = _f64(s["grad"])
    if case["activation"] != "none":
        pre = _f64(s["pre"]).requires_grad_()
        dz, = torch.autograd.grad(_exact_activation(pre, case["activation"]), pre, dz)
    dx = torch.cat([dz[a:b] @ w[e].T for e, (a, b) in enumerate(spans)])
    dw = torch.stack([x[a:b].T @ dz[a:b] for a, b in spans])
    out = {"dx": dx, "dw": dw.reshape(s["weight"].shape)}
    if case["bias"]:
        db = torch.stack([dz[a:b].sum(0) for a, b in spans])
        out["dbias"] = db.reshape(-1) if case["op"] == "linear" else db
    return out
