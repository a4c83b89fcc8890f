"""Dense layers in 8-bit integers with a scale for each token and each channel, layer normalisation, and activations
that are kept in 8 bits for the backward pass, as timed cases: the plain forms in elementary torch operations, and
the calls of ``approxtrain_amd`` that a user makes instead."""
import math

import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_EPSILON = 1e-3


# ---- cases ------------------------------------------------------------------------------------------

def _serve(name, rows, fan_in, units, dtype, relu):
    return {"name": name, "op": "serve", "rows": rows, "fan_in": fan_in, "units": units, "dtype": dtype, "relu": relu}


# (A rectifier between the products would let a sum near zero through or not by its last bit, and every
# gradient behind it with it: the training steps here are of layers without one.)
def _train(name, rows, fan_in, units, dtype, kernel_dtype):
    return {"name": name, "op": "train", "rows": rows, "fan_in": fan_in, "units": units, "dtype": dtype,
            "kernel_dtype": kernel_dtype}


def _norm(name, rows, cols, dtype, way):
    return {"name": name, "op": "norm", "rows": rows, "cols": cols, "dtype": dtype, "way": way}


def _act(name, rows, cols, dtype, kind):
    return {"name": name, "op": "act", "rows": rows, "cols": cols, "dtype": dtype, "kind": kind}


def listed():
    return [
        # one token through a square layer whose weights lie there in 8 bits: a latency
        _serve("serve_token", 1, 4096, 4096, "bfloat16", False),
        # a few sequences' next tokens, odd extents, with bias and rectifier
        _serve("serve_few_odd", 13, 2051, 1003, "float32", True),
        # inference over a whole batch of prompts
        _serve("serve_batch", 4096, 4096, 4096, "bfloat16", True),
        # the training step of LeNet-300-100's first layer
        _train("train_lenet300", 128, 784, 300, "float32", "float32"),
        # a projection of the encoder block (32 sequences of 256 positions, depth 512)
        _train("train_projection", 8192, 512, 512, "float32", "float32"),
        # the largest training step: mixed precision, 32-bit weights under 16-bit activations
        _train("train_4096", 4096, 4096, 4096, "bfloat16", "float32"),
        # one sequence of the encoder normalised for inference: a latency
        _norm("norm_sequence", 256, 512, "float32", "serve"),
        # a training step over a ragged batch of odd width
        _norm("norm_odd", 1999, 1027, "float16", "train"),
        # a wide model's training step whose input is kept in 8 bits
        _norm("norm_large_kept", 16384, 4096, "bfloat16", "kept"),
        # the hidden layer of the encoder's feed-forward half, four times its depth
        _act("act_encoder", 8192, 2048, "float32", "gelu"),
        # odd extents
        _act("act_odd", 1999, 1027, "bfloat16", "swish"),
        # a wide model's hidden layer
        _act("act_large", 16384, 4096, "bfloat16", "gelu"),
    ]


def _log_int(rng, lo, hi):
    """An integer from [lo, hi], spread over the logarithm; about a third of them multiples of 32."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v >= 64 and rng.random() < 0.35:
        v = v // 32 * 32
    return min(max(v, lo), hi)


def draw(rng):
    while True:
        op = rng.choice(("serve", "serve", "train", "train", "norm", "norm", "act"))
        dtype = rng.choice(("float32", "bfloat16", "bfloat16", "float16"))
        if op == "serve":
            rows = _log_int(rng, 1, 64) if rng.random() < 0.5 else _log_int(rng, 64, 8192)
            c = _serve("", rows, _log_int(rng, 32, 8192), _log_int(rng, 10, 8192), dtype, rng.random() < 0.5)
        elif op == "train":
            c = _train("", _log_int(rng, 8, 16384), _log_int(rng, 32, 8192), _log_int(rng, 10, 8192), dtype,
                       rng.choice(("float32", dtype)))
        elif op == "norm":
            c = _norm("", _log_int(rng, 1, 16384), _log_int(rng, 16, 16384), dtype, rng.choice(("serve", "train", "kept")))
        else:
            c = _act("", _log_int(rng, 1, 16384), _log_int(rng, 16, 16384), dtype, rng.choice(("gelu", "swish")))
        del c["name"]
        w = work(c)
        if w["bytes"] <= 5.4e8 and w["flops"] <= 4.2e11:
            return c


# ---- what a user's program holds before the call ----------------------------------------------------

def _activations(gen, rows, cols, dtype):
    """Normal values whose channels differ in scale, a few of them by much."""
    channel = torch.exp(torch.randn(cols, device="cuda", generator=gen) * 0.5)
    return (torch.randn((rows, cols), device="cuda", generator=gen) * channel).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    dtype = _TYPES[case["dtype"]]
    if case["op"] in ("serve", "train"):
        rows, fan_in, units = case["rows"], case["fan_in"], case["units"]
        train = case["op"] == "train"
        s["x"] = _activations(gen, rows, fan_in, dtype).requires_grad_(train)
        kernel = torch.randn((fan_in, units), device="cuda", generator=gen) / math.sqrt(fan_in)
        kernel = kernel.to(_TYPES[case["kernel_dtype"] if train else case["dtype"]])
        s["bias"] = (torch.randn(units, device="cuda", generator=gen) * 0.1).requires_grad_(train)
        if train:
            s["kernel"] = kernel.requires_grad_()
            s["dy"] = (torch.randn((rows, units), device="cuda", generator=gen) * 1e-2).to(dtype)
        elif own:  # a server keeps the weights as they are multiplied: 8 bits here, the same numbers in 32 there
            from approxtrain_amd import functors
            s["weights"] = functors.int8_quantize(kernel, axis=0)
        else:
            s["weights"], s["kernel"] = _codes(kernel.t()), kernel
        return s
    rows, cols = case["rows"], case["cols"]
    train = case["op"] == "act" or case["way"] != "serve"
    s["x"] = _activations(gen, rows, cols, dtype).requires_grad_(train)
    if case["op"] == "norm":
        s["gamma"] = (1 + 0.1 * torch.randn(cols, device="cuda", generator=gen)).requires_grad_(train)
        s["beta"] = (0.1 * torch.randn(cols, device="cuda", generator=gen)).requires_grad_(train)
    if train:
        s["dy"] = (torch.randn((rows, cols), device="cuda", generator=gen) * 1e-2).to(dtype)
    return s


# ---- the plain forms ----------------------------------------------------------------------------------

def _codes(v):
    """(codes, scales) of ``v``'s rows as 8-bit integers: v * (127 / largest), rounded to the nearest integer, ties to
    even, from the exact product (in 64 bits: values next to a border, and quotients that are rounded to 32 bits once)."""
    v = v.double()
    largest = v.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -119)
    return torch.round(v * (127 / largest).float()).float(), (largest / 127).float()


def _plain_train(s):
    x, kernel, bias, dy = s["x"], s["kernel"], s["bias"], s["dy"]
    (qx, sx), (qw, sw) = _codes(x), _codes(kernel.t())
    out = (torch.matmul(qx, qw.t()) * sx * sw.t() + bias.float()).to(x.dtype)
    g = dy.float()
    qv, sv = _codes(g * sw.t())
    dx = (torch.matmul(qv, qw) * sv).to(x.dtype)
    qu, su = _codes((g * sx).t())
    dw = (torch.matmul(qx.t(), qu.t()) * su.t()).to(kernel.dtype)
    return out, dx, dw, g.sum(0).to(bias.dtype)


def _plain_norm(s):
    x, gamma, beta, way = s["x"], s["gamma"], s["beta"], s["case"]["way"]
    f = x.float()
    mean = f.mean(-1, keepdim=True)
    rstd = torch.rsqrt((f - mean).square().mean(-1, keepdim=True) + _EPSILON)
    y = ((f - mean) * rstd * gamma + beta).to(x.dtype)
    if way == "serve":
        return y
    if way == "kept":
        q, scale = _codes(x)
        f = q * scale
    normal, dy = (f - mean) * rstd, s["dy"].float()
    g = dy * gamma
    dx = rstd * (g - g.mean(-1, keepdim=True) - normal * (g * normal).mean(-1, keepdim=True))
    return y, dx.to(x.dtype), (dy * normal).sum(0), dy.sum(0)


def _plain_act(s):
    x, kind = s["x"], s["case"]["kind"]
    f = x.float()
    q, scale = _codes(x)
    kept = q * scale
    if kind == "gelu":
        y = f * (0.5 * torch.erfc(f * -math.sqrt(0.5)))
        slope = 0.5 * torch.erfc(kept * -math.sqrt(0.5)) + kept * torch.exp(kept * kept * -0.5) * (1 / math.sqrt(2 * math.pi))
    else:
        y = f / (1 + torch.exp(-f))
        g = 1 / (1 + torch.exp(-kept))
        slope = g + kept * g * (1 - g)
    return y.to(x.dtype), (s["dy"].float() * slope).to(x.dtype)


def _plain(s):
    case = s["case"]
    with torch.no_grad():
        if case["op"] == "serve":
            (qx, sx), (qw, sw) = _codes(s["x"]), s["weights"]
            z = torch.matmul(qx, qw.t()) * sx * sw.t() + s["bias"].float()
            return (torch.relu(z) if case["relu"] else z).to(s["x"].dtype)
        return {"train": _plain_train, "norm": _plain_norm, "act": _plain_act}[case["op"]](s)


# ---- the framework's calls ------------------------------------------------------------------------------

def _own(s):
    from approxtrain_amd import functors, math_ops
    case = s["case"]
    if case["op"] == "serve":
        return functors.int8_linear(s["x"], s["weights"], bias=s["bias"], activation="relu" if case["relu"] else None)
    if case["op"] == "train":
        out = math_ops.lineari8(s["x"], s["kernel"], s["bias"])
        return (out.detach(),) + torch.autograd.grad(out, [s["x"], s["kernel"], s["bias"]], s["dy"])
    if case["op"] == "norm":
        if case["way"] == "serve":
            return functors.layer_norm(s["x"], s["gamma"], s["beta"], epsilon=_EPSILON)
        y = math_ops.layernorm(s["x"], s["gamma"], s["beta"], epsilon=_EPSILON, keep_bits=8 if case["way"] == "kept" else None)
        return (y.detach(),) + torch.autograd.grad(y, [s["x"], s["gamma"], s["beta"]], s["dy"])
    y = math_ops.activationi8(s["x"], case["kind"])
    return (y.detach(),) + torch.autograd.grad(y, [s["x"]], s["dy"])


def run(state):
    """One pass: a layer's output, its training step, or a normalisation's or an activation's."""
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------

def work(case):
    b = 4 if case["dtype"] == "float32" else 2
    if case["op"] in ("norm", "act"):
        n = case["rows"] * case["cols"]
        if case["op"] == "act":
            return {"bytes": 4 * b * n, "flops": 30 * n}
        if case["way"] == "serve":
            return {"bytes": 2 * b * n + 8 * case["cols"], "flops": 8 * n}
        return {"bytes": 4 * b * n + 16 * case["cols"], "flops": 22 * n}
    rows, fan_in, units = case["rows"], case["fan_in"], case["units"]
    macs = rows * fan_in * units
    if case["op"] == "serve":
        return {"bytes": b * rows * (fan_in + units) + fan_in * units + 8 * units, "flops": 2 * macs}
    k = 4 if case["kernel_dtype"] == "float32" else 2
    return {"bytes": 2 * b * rows * (fan_in + units) + 2 * k * fan_in * units + 8 * units, "flops": 6 * macs}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------

def _exact_int8(v, axis):
    """Integers and scale (a number of 32 bits each) that stand for ``v`` (64 bits) along ``axis``."""
    top = torch.maximum(v.abs().max(axis, keepdim=True).values, torch.full((), 2.0 ** -119, dtype=torch.float64, device=v.device))
    per_unit, unit = (127.0 / top).float().double(), (top / 127.0).float().double()
    product = v * per_unit
    below = torch.floor(product)
    rest = product - below
    up = (rest > 0.5) | ((rest == 0.5) & (torch.remainder(below, 2) == 1))
    return below + up, unit


def _rounded(v):
    return v.float().double()


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].detach().double()
    if case["op"] in ("serve", "train"):
        w, bias = s["kernel"].detach().double(), s["bias"].detach().double()
        (ix, ux), (iw, uw) = _exact_int8(x, 1), _exact_int8(w, 0)
        z = (ix @ iw) * (ux * uw) + bias
        if case["op"] == "serve":
            return z.clamp(min=0) if case["relu"] else z
        dy = s["dy"].double()
        # (what the gradient is multiplied by before it becomes integers is rounded to 32 bits: part of the definition)
        ia, ua = _exact_int8(_rounded(dy * uw), 1)
        ib, ub = _exact_int8(_rounded(dy * ux), 0)
        return z, (ia @ iw.t().contiguous()) * ua, (ix.t().contiguous() @ ib) * ub, dy.sum(0)
    if case["op"] == "norm":
        gamma, beta = s["gamma"].detach().double(), s["beta"].detach().double()
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        sigma = torch.sqrt(var + _EPSILON)
        y = (x - mean) / sigma * gamma + beta
        if case["way"] == "serve":
            return y
        if case["way"] == "kept":
            i, u = _exact_int8(x, 1)
            x = i * u
        h, dy = (x - mean) / sigma, s["dy"].double()
        t = dy * gamma / sigma
        n = x.shape[1]
        dx = t - t.sum(1, keepdim=True) / n - h * ((t * h).sum(1, keepdim=True) / n)
        return y, dx, (dy * h).sum(0), dy.sum(0)
    i, u = _exact_int8(x, 1)
    if case["kind"] == "gelu":
        def value(t):
            return t * torch.special.ndtr(t)

        def slope(t):
            return torch.special.ndtr(t) + t * torch.exp(-t * t / 2) / math.sqrt(2 * math.pi)
    else:
        def value(t):
            return t * torch.sigmoid(t)

        def slope(t):
            return torch.sigmoid(t) * (1 + t * torch.sigmoid(-t))
    return value(x), s["dy"].double() * slope(i * u)
