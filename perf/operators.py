"""Training and serving of dense layers in microscaled 4-bit floating point (MXFP4: blocks of 32 e2m1
elements along the reduction axis with one power-of-two scale each), and the AdamW step that updates such
layers' weights, as timed cases: the plain forms in elementary torch operations, and the calls of
``approxtrain_amd`` that a user makes instead."""
import math
import random

import torch
import torch.nn.functional as F

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ---- cases ------------------------------------------------------------------------------------------

def _quantize(name, rows, cols, dtype, way):
    return {"name": name, "op": "quantize", "rows": rows, "cols": cols, "dtype": dtype, "way": way}


def _serve(name, rows, fan_in, units, dtype, relu):
    return {"name": name, "op": "serve", "rows": rows, "fan_in": fan_in, "units": units, "dtype": dtype, "relu": relu}


# (A rectifier between the products would let a sum near zero through or not by its last bit, and every
# gradient behind it with it: the training steps here are of layers without one.)
def _train(name, rows, fan_in, units, dtype, kernel_dtype):
    return {"name": name, "op": "train", "rows": rows, "fan_in": fan_in, "units": units, "dtype": dtype,
            "kernel_dtype": kernel_dtype}


def _adamw(name, tensors, bits, dtype, grad_dtype, clip):
    return {"name": name, "op": "adamw", "tensors": tensors, "bits": bits, "dtype": dtype, "grad_dtype": grad_dtype,
            "clip": clip}


def listed():
    return [
        # a batch of flattened images made 4-bit for the first layer of LeNet-300-100: a latency
        _quantize("quantize_lenet300", 128, 784, "float32", "rows"),
        # activations of odd extents, as the second operand of a weight gradient: blocks down the columns
        _quantize("quantize_odd_columns", 1999, 1027, "float16", "columns"),
        # the activations of a wide layer's training step: both directions from one reading
        _quantize("quantize_both_large", 8192, 4096, "bfloat16", "both"),
        # one token through a square layer whose weights lie there in 4 bits
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
        # the optimizer's step of LeNet-300-100: six tensors, a latency
        _adamw("adamw_lenet300", "stack:784,300,100,10", 32, "float32", "float32", False),
        # ... of ResNet-50's convolutions and biases, states in 8 bits
        _adamw("adamw_resnet50_8bit", "resnet50", 8, "float32", "float32", True),
        # ... of a deep encoder with 16-bit gradients, states in 32 bits
        _adamw("adamw_encoder", "encoder:24,1024", 32, "float32", "bfloat16", True),
    ]


def _log_int(rng, lo, hi):
    """An integer from [lo, hi], spread over the logarithm; about a third of them multiples of 32."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v >= 64 and rng.random() < 0.35:
        v = v // 32 * 32
    return min(max(v, lo), hi)


def draw(rng):
    while True:
        op = rng.choice(("quantize", "serve", "serve", "train", "train", "adamw"))
        dtype = rng.choice(("float32", "bfloat16", "bfloat16", "float16"))
        if op == "quantize":
            c = _quantize("", _log_int(rng, 1, 16384), _log_int(rng, 16, 16384), dtype, rng.choice(("rows", "columns", "both")))
        elif op == "serve":
            rows = _log_int(rng, 1, 64) if rng.random() < 0.5 else _log_int(rng, 64, 8192)
            c = _serve("", rows, _log_int(rng, 32, 8192), _log_int(rng, 10, 8192), dtype, rng.random() < 0.5)
        elif op == "train":
            c = _train("", _log_int(rng, 8, 16384), _log_int(rng, 32, 8192), _log_int(rng, 10, 8192), dtype,
                       rng.choice(("float32", dtype)))
        else:
            c = _adamw("", "mixed:%d,%d,%d,%d" % (_log_int(rng, 1, 200), _log_int(rng, 1, 512), _log_int(rng, 1024, 1 << 22),
                                                  rng.randrange(1 << 20)),
                       rng.choice((32, 8)), rng.choice(("float32", "float32", "bfloat16")), rng.choice(("float32", "bfloat16")),
                       rng.random() < 0.5)
        del c["name"]
        w = work(c)
        if w["bytes"] <= 8.0e9 and w["flops"] <= 4.2e11:
            return c


# ---- the tensors of an optimizer's step ---------------------------------------------------------------

_BLOCK = 256  # elements of an optimizer state that share one scale


def _sizes(case):
    kind, _, rest = case["tensors"].partition(":")
    if kind == "stack":  # dense layers of these widths, each a kernel and a bias
        widths = [int(v) for v in rest.split(",")]
        return [n for a, b in zip(widths, widths[1:]) for n in (a * b, b)]
    if kind == "resnet50":  # bottleneck stages: 1x1, 3x3 and 1x1 convolutions with biases, then the classifier
        sizes, c = [7 * 7 * 3 * 64, 64], 64
        for width, blocks in ((64, 3), (128, 4), (256, 6), (512, 3)):
            for b in range(blocks):
                convs = [(1, c, width), (3, width, width), (1, width, 4 * width)] + ([(1, c, 4 * width)] if b == 0 else [])
                sizes += [n for k, i, o in convs for n in (k * k * i * o, o)]
                c = 4 * width
        return sizes + [2048 * 1000, 1000]
    if kind == "encoder":  # blocks of four projections, each a kernel and a bias
        blocks, d = [int(v) for v in rest.split(",")]
        return [d * d, d] * (4 * blocks)
    count, lo, hi, seed = [int(v) for v in rest.split(",")]
    r = random.Random(seed)
    return [int(math.exp(r.uniform(math.log(lo), math.log(hi)))) for _ in range(count)]


def _layout(case):
    """(size, start in the flat buffer) of each tensor: every one starts on a block of its own."""
    at, got = 0, []
    for n in _sizes(case):
        got.append((n, at))
        at += -(-n // _BLOCK) * _BLOCK
    return got, at


_HYPER = {"lr": 1e-3, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8, "weight_decay": 0.01, "step": 100}


# ---- what a user's program holds before the call ----------------------------------------------------

def _activations(gen, rows, cols, dtype):
    """Normal values whose channels differ in scale, a few of them by much."""
    channel = torch.exp(torch.randn(cols, device="cuda", generator=gen) * 0.5)
    return (torch.randn((rows, cols), device="cuda", generator=gen) * channel).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "quantize":
        s["x"] = _activations(gen, case["rows"], case["cols"], _TYPES[case["dtype"]])
    elif case["op"] in ("serve", "train"):
        rows, fan_in, units, dtype = case["rows"], case["fan_in"], case["units"], _TYPES[case["dtype"]]
        train = case["op"] == "train"
        s["x"] = _activations(gen, rows, fan_in, dtype).requires_grad_(train)
        kernel = torch.randn((fan_in, units), device="cuda", generator=gen) / math.sqrt(fan_in)
        kernel = kernel.to(_TYPES[case["kernel_dtype"] if train else case["dtype"]])
        s["bias"] = (torch.randn(units, device="cuda", generator=gen) * 0.1).requires_grad_(train)
        if train:
            s["kernel"] = kernel.requires_grad_()
            s["dy"] = (torch.randn((rows, units), device="cuda", generator=gen) * 1e-2).to(dtype)
        elif own:  # a server keeps the weights as they are multiplied: 4 bits here, their values in 32 there
            from approxtrain_amd import functors
            s["weights"] = functors.mxfp4_quantize(kernel, axis=0)
        else:
            s["weights"], s["kernel"] = _mx_values(kernel.t().contiguous()), kernel
    else:
        layout, total = _layout(case)
        flat = {"p": torch.zeros(total, device="cuda", dtype=_TYPES[case["dtype"]]),
                "g": torch.zeros(total, device="cuda", dtype=_TYPES[case["grad_dtype"]])}
        if case["bits"] == 32:
            flat["m"], flat["v"] = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
        else:
            flat["m"] = torch.zeros(total, device="cuda", dtype=torch.uint8)
            flat["v"] = torch.zeros(total, device="cuda", dtype=torch.uint8)
            flat["m_scale"] = torch.zeros(total // _BLOCK, device="cuda")
            flat["v_scale"] = torch.zeros(total // _BLOCK, device="cuda")
        used = torch.zeros(total, dtype=torch.bool, device="cuda")
        for n, at in layout:
            used[at:at + n] = True
        # gradients whose size varies from one neuron to the next, states of some steps' history
        flat["p"].copy_(torch.randn(total, device="cuda", generator=gen) * 0.05 * used)
        size = torch.exp(torch.randn(total // _BLOCK, device="cuda", generator=gen) - 6).repeat_interleave(_BLOCK) * used
        flat["g"].copy_(torch.randn(total, device="cuda", generator=gen) * size)
        m = torch.randn(total, device="cuda", generator=gen) * size * 0.3
        v = (torch.rand(total, device="cuda", generator=gen) + 0.1) * size * size
        if case["bits"] == 32:
            flat["m"].copy_(m), flat["v"].copy_(v)
        else:
            (flat["m"][:], flat["m_scale"][:]), (flat["v"][:], flat["v_scale"][:]) = _encode_m(m), _encode_r(v.sqrt())
        s["flat"] = flat
        s["grad_scale"] = torch.full((1,), 0.7, device="cuda") if case["clip"] else None
        if own:  # the optimizer's states lie as here: one buffer, every tensor from a block of its own on
            from approxtrain_amd import functors
            s["params"], s["grads"] = ([flat[k][at:at + n] for n, at in layout] for k in ("p", "g"))
            s["state"] = functors.AdamWState(s["params"], case["bits"])
            for k in ("m", "v", "m_scale", "v_scale"):
                if k in flat:
                    getattr(s["state"], k).copy_(flat[k])
    return s


# ---- the plain forms ----------------------------------------------------------------------------------

def _mx_values(x):
    """The values that ``x`` has in MXFP4 with blocks along its last axis, in 32 bits: scale 2^(e - 2) with
    e the exponent of the block's largest magnitude, elements rounded to nearest-even and saturated."""
    rows, cols = x.shape
    f = F.pad(x.float(), (0, -cols % 32)).reshape(rows, -1, 32)
    largest = (f.view(torch.int32) & 0x7FFFFFFF).amax(-1, keepdim=True)
    code = ((largest >> 23) - 2).clamp(min=0)
    scale = torch.where(code > 0, code << 23, torch.full_like(code, 1 << 22)).view(torch.float32)  # 2^(code - 127)
    inverse = ((254 - code) << 23).view(torch.float32)                                             # 2^(127 - code)
    t = f * inverse
    a = t.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = torch.clamp(torch.round(a / step) * step, max=6.0)
    values = torch.where(largest >= 0x7F800000, torch.nan, torch.copysign(q, t) * scale)
    return values.reshape(rows, -1)[:, :cols]


def _dense(values_x, values_w, bias, relu, dtype):
    z = torch.matmul(values_x, values_w.t()) + bias.float()
    return (torch.relu(z) if relu else z).to(dtype)


# 8-bit codes of optimizer states: magnitudes relative to the block's largest, the upper bits of their
# 32-bit form.  First moments: sign, 4 exponent bits, 3 of mantissa.  Roots of second moments: 4 and 4.
_M_SHIFT, _M_BASE = 20, 889
_R_SHIFT, _R_BASE = 19, 1777


def _codes(t, shift, base):
    bits = t.view(torch.int32)
    return ((bits + ((1 << (shift - 1)) - 1) + ((bits >> shift) & 1)) >> shift) - base


def _relative(x):
    blocks = x.reshape(-1, _BLOCK)
    scale = blocks.abs().amax(-1, keepdim=True)
    return torch.where(scale > 0, blocks.abs() / scale, 0.0), scale


def _encode_m(m):
    t, scale = _relative(m)
    smallest = torch.tensor([(_M_BASE + 1) << _M_SHIFT], dtype=torch.int32, device=m.device).view(torch.float32)
    c = torch.where(t < smallest * 0.5, 0, _codes(t, _M_SHIFT, _M_BASE).clamp(1, 127))
    c = torch.where(m.reshape(-1, _BLOCK) < 0, c + 128, c)
    return c.to(torch.uint8).reshape(-1), scale.reshape(-1)


def _encode_r(r):
    t, scale = _relative(r)
    c = torch.where(t > 0, _codes(t, _R_SHIFT, _R_BASE).clamp(1, 255), 0)
    return c.to(torch.uint8).reshape(-1), scale.reshape(-1)


def _decode(code, scale, shift, base):
    magnitude = torch.where(code > 0, (code.to(torch.int32) + base) << shift, 0).view(torch.float32)
    return (magnitude.reshape(-1, _BLOCK) * scale.reshape(-1, 1)).reshape(-1)


def _decode_m(code, scale):
    magnitude = _decode(code & 127, scale, _M_SHIFT, _M_BASE)
    return torch.where(code >= 128, -magnitude, magnitude)


def _decode_r(code, scale):
    return _decode(code, scale, _R_SHIFT, _R_BASE)


def _plain_adamw(s):
    """One step over the flat buffers, so that each operation runs over all tensors at once."""
    f, h, bits = s["flat"], _HYPER, s["case"]["bits"]
    g = f["g"].float()
    if s["grad_scale"] is not None:
        g = g * s["grad_scale"]
    m = f["m"] if bits == 32 else _decode_m(f["m"], f["m_scale"])
    v = f["v"] if bits == 32 else _decode_r(f["v"], f["v_scale"]).square()
    m = m * h["beta1"] + g * (1 - h["beta1"])
    v = v * h["beta2"] + (g * (1 - h["beta2"])) * g
    r = v.sqrt()
    denominator = r / math.sqrt(1 - h["beta2"] ** h["step"]) + h["eps"]
    update = (m / denominator) * (h["lr"] / (1 - h["beta1"] ** h["step"]))
    f["p"].copy_(f["p"].float() * (1 - h["lr"] * h["weight_decay"]) - update)
    if bits == 32:
        f["m"].copy_(m), f["v"].copy_(v)
        return f["p"], f["m"], f["v"]
    (m_code, m_scale), (r_code, r_scale) = _encode_m(m), _encode_r(r)
    f["m"].copy_(m_code), f["m_scale"].copy_(m_scale), f["v"].copy_(r_code), f["v_scale"].copy_(r_scale)
    return f["p"], _decode_m(f["m"], f["m_scale"]), _decode_r(f["v"], f["v_scale"])


def _plain(s):
    case = s["case"]
    if case["op"] == "quantize":
        x = s["x"]
        rows = _mx_values(x).to(x.dtype) if case["way"] != "columns" else None
        columns = _mx_values(x.t().contiguous()).to(x.dtype) if case["way"] != "rows" else None
        return [v for v in (rows, columns) if v is not None]
    if case["op"] == "serve":
        return _dense(_mx_values(s["x"]), s["weights"], s["bias"], case["relu"], s["x"].dtype)
    if case["op"] == "train":
        with torch.no_grad():
            x, kernel, bias, dy = s["x"], s["kernel"], s["bias"], s["dy"]
            out = _dense(_mx_values(x), _mx_values(kernel.t().contiguous()), bias, False, x.dtype)
            dx = torch.matmul(_mx_values(dy), _mx_values(kernel).t()).to(x.dtype)
            dw = torch.matmul(_mx_values(x.t().contiguous()), _mx_values(dy.t().contiguous()).t()).to(kernel.dtype)
            return out, dx, dw, dy.float().sum(0).to(bias.dtype)
    return _plain_adamw(s)


# ---- the framework's calls ------------------------------------------------------------------------------

def _own(s):
    from approxtrain_amd import functors, math_ops
    case = s["case"]
    if case["op"] == "quantize":
        x = s["x"]
        if case["way"] == "both":
            parts = functors.mxfp4_quantize_both(x)
        else:
            parts = [functors.mxfp4_quantize(x, axis=-1 if case["way"] == "rows" else 0)]
        return [functors.mxfp4_dequantize(q, x.dtype) for q in parts]
    if case["op"] == "serve":
        return functors.mxfp4_linear(s["x"], s["weights"], bias=s["bias"], activation="relu" if case["relu"] else None)
    if case["op"] == "train":
        out = math_ops.linearmx(s["x"], s["kernel"], s["bias"])
        return (out.detach(),) + torch.autograd.grad(out, [s["x"], s["kernel"], s["bias"]], s["dy"])
    state = s["state"]
    functors.adamw_step(state, s["grads"], grad_scale=s["grad_scale"], **_HYPER)
    if case["bits"] == 32:
        return s["flat"]["p"], state.m, state.v
    return s["flat"]["p"], state.first_moments(), state.second_roots()


def run(state):
    """One pass: the 4-bit values of a tensor, a layer's output, a layer's training step, or an optimizer's step."""
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------

def work(case):
    b = 4 if case.get("dtype") == "float32" else 2
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": n * b * (3 if case["way"] == "both" else 2), "flops": 0}
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        state = 16 if case["bits"] == 32 else 4 * (1 + 4 / _BLOCK) + 8  # (8 bits: their values are written out too)
        return {"bytes": n * (2 * b + (4 if case["grad_dtype"] == "float32" else 2) + state), "flops": 14 * n}
    rows, fan_in, units = case["rows"], case["fan_in"], case["units"]
    macs = rows * fan_in * units
    if case["op"] == "serve":
        return {"bytes": b * rows * (fan_in + units) + 17 * fan_in * units / 32 + 4 * units, "flops": 2 * macs}
    k = 4 if case["kernel_dtype"] == "float32" else 2
    return {"bytes": 2 * b * rows * (fan_in + units) + 2 * k * fan_in * units + 8 * units, "flops": 6 * macs}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------

def _power_of_two(n):
    return ((n.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_mx(x, axis):
    """Values of ``x`` (64 bits) in MXFP4 with blocks along ``axis``: the nearest of the format's numbers."""
    x = x.movedim(axis, -1)
    n = x.shape[-1]
    blocks = torch.cat([x, x.new_zeros(x.shape[:-1] + (-n % 32,))], -1).unflatten(-1, (-1, 32))
    _, e = torch.frexp(blocks.abs().amax(-1, keepdim=True))  # largest = f * 2^e, f in [0.5, 1)
    scale = _power_of_two((e - 3).clamp(min=-127))
    numbers = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    middle = (numbers[1:] + numbers[:-1]) / 2
    up = torch.tensor([0, 1, 0, 1, 0, 1, 0], dtype=torch.bool, device=x.device)  # a tie goes to the even code
    border = torch.where(up, middle, torch.nextafter(middle, torch.full_like(middle, 9.0)))
    q = numbers[torch.bucketize((blocks.abs() / scale).contiguous(), border, right=True)]
    return (torch.sign(blocks) * q * scale).flatten(-2)[..., :n].movedim(-1, axis)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        x = s["x"].double()
        return [_exact_mx(v, 1) for way, v in (("rows", x), ("columns", x.t())) if case["way"] in (way, "both")]
    if case["op"] == "adamw":
        return _exact_adamw(s)
    x, w, bias = (s[k].detach().double() for k in ("x", "kernel", "bias"))
    z = _exact_mx(x, 1) @ _exact_mx(w, 0) + bias
    if case["op"] == "serve":
        return z.clamp(min=0) if case["relu"] else z
    dy = s["dy"].double()
    return z, _exact_mx(dy, 1) @ _exact_mx(w, 1).t(), _exact_mx(x, 0).t() @ _exact_mx(dy, 0), dy.sum(0)


def _exact_adamw(s):
    f, h, case = s["flat"], _HYPER, s["case"]
    g = f["g"].double() * (1.0 if s["grad_scale"] is None else s["grad_scale"].double())
    if case["bits"] == 32:
        m, v = f["m"].double(), f["v"].double()
    else:
        byte = f["m"].to(torch.int64)
        m = _exact_minifloat(byte % 128, 3) * f["m_scale"].double().repeat_interleave(_BLOCK) * (1 - 2.0 * (byte >= 128))
        v = (_exact_minifloat(f["v"].to(torch.int64), 4) * f["v_scale"].double().repeat_interleave(_BLOCK)) ** 2
    m = h["beta1"] * m + (1 - h["beta1"]) * g
    v = h["beta2"] * v + (1 - h["beta2"]) * g * g
    m_hat, v_hat = m / (1 - h["beta1"] ** h["step"]), v / (1 - h["beta2"] ** h["step"])
    p = f["p"].double()
    p = p - h["lr"] * h["weight_decay"] * p - h["lr"] * m_hat / (v_hat.sqrt() + h["eps"])
    # (a state that is rounded to 8 bits steps where the last bit of 32 decides: no value of its own in 64)
    return (p, m, v) if case["bits"] == 32 else (p, None, None)


def _exact_minifloat(code, mantissa_bits):
    """The number a code stands for, 1 the largest: code 0 is 0, others count down from 2^0 in binades of 2^mantissa_bits."""
    below = (127 if mantissa_bits == 3 else 255) - code
    steps = 1 << mantissa_bits
    binade = torch.div(below + steps - 1, steps, rounding_mode="floor")
    within = binade * steps - below
    return torch.where(code > 0, _power_of_two(-binade) * (1 + within.double() / steps), 0.0)
