"""The definitions of the row operators and of the 8-bit products in 64 bits, for the tests."""
import math

import torch

U = 2.0 ** -24  # a rounding to 32 bits


def half_step(dtype):
    """A rounding to ``dtype``, relative."""
    return torch.finfo(dtype).eps / 2


def int8(v, axis=-1):
    """(codes, scale) of ``v`` along ``axis``: codes as whole numbers in 64 bits, the scale a number of 32."""
    v = v.double()
    largest = v.abs().amax(axis, keepdim=True).clamp(min=2.0 ** -119)
    return torch.round(v * (127.0 / largest).float().double()), (largest / 127.0).float().double()


def int8_values(v, axis=-1):
    q, s = int8(v, axis)
    return q * s


def gelu(x):
    return 0.5 * x * torch.erfc(-x / math.sqrt(2.0))


def gelu_slope(x):
    return 0.5 * torch.erfc(-x / math.sqrt(2.0)) + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)


def swish(x):
    return x * torch.sigmoid(x)


def swish_slope(x):
    s = torch.sigmoid(x)
    return s + x * s * (1 - s)


ACTIVATIONS = {"gelu": (gelu, gelu_slope), "swish": (swish, swish_slope)}


def layer_norm(x, gamma, beta, epsilon, grad=None, kept=None):
    """y, or (y, dx, dgamma, dbeta) for ``grad``; ``kept``: what stands in for x in the gradients."""
    x = x.double()
    gamma = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if gamma is None else gamma.double()
    beta = torch.zeros_like(gamma) if beta is None else beta.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + epsilon)
    y = (x - mean) * rstd * gamma + beta
    if grad is None:
        return y
    h, g = ((x if kept is None else kept.double()) - mean) * rstd, grad.double()
    t = g * gamma
    dx = rstd * (t - t.mean(-1, keepdim=True) - h * (t * h).mean(-1, keepdim=True))
    lead = tuple(range(x.dim() - 1))
    return y, dx, (g * h).sum(lead), g.sum(lead)


def layer_norm_tolerances(x, gamma, beta, epsilon, grad=None, kept=None):
    """How far the results of ``layer_norm`` may be off in 32-bit arithmetic, before they are rounded to their types.

    A lane adds up at most cols / 1024 + 16 values of a row, the lanes' sums meet in at most 6 + 16 steps and a division
    follows: n roundings.  mean is off by e = n u mean|x|; the squares about it by n + 4 roundings and, in the
    second order, by e^2; 1 / sqrt halves a relative error and adds three roundings.  Over the rows a lane adds at most
    rows / 64, the workgroups' sums at most 16 + 5 more, 16 in LDS."""
    x = x.double()
    cols, rows = x.shape[-1], x.numel() // x.shape[-1]
    gamma = torch.ones(cols, dtype=torch.float64, device=x.device) if gamma is None else gamma.double()
    beta = torch.zeros_like(gamma) if beta is None else beta.double()
    n = (cols / 1024 + 44) * U
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + epsilon)
    e = n * x.abs().mean(-1, keepdim=True)
    r = (n + 4 * U + (e * rstd) ** 2) / 2 + 3 * U

    def normal(v):
        h = (v - mean) * rstd
        return h, rstd * (e + U * v.abs()) + h.abs() * (r + 2 * U)

    h, eh = normal(x)
    y = gamma.abs() * eh + 2 * U * ((gamma * h).abs() + beta.abs())
    if grad is None:
        return y * 1.01
    if kept is not None:
        h, eh = normal(kept.double())
    g = grad.double()
    t = g * gamma
    mt, dot = t.mean(-1, keepdim=True), (t * h).mean(-1, keepdim=True)
    e_mt = (n + U) * t.abs().mean(-1, keepdim=True)
    e_dot = (t.abs() * eh).mean(-1, keepdim=True) + (n + 2 * U) * (t * h).abs().mean(-1, keepdim=True)
    size = t.abs() + mt.abs() + (h * dot).abs()
    dx = rstd * (e_mt + eh * dot.abs() + h.abs() * e_dot + (4 * U + r + 2 * U) * size)
    lead = tuple(range(x.dim() - 1))
    m = (rows / 64 + 80) * U
    return y * 1.01, dx * 1.01, ((g.abs() * eh).sum(lead) + m * (g * h).abs().sum(lead)) * 1.01, m * g.abs().sum(lead) * 1.01


def activation_tolerances(kind, x, kept):
    """The same of ``ACTIVATIONS[kind]`` at x and of its slope at ``kept``.

    gelu: the tail Phi(-|x|) is u P(u) e.  P fits to 1.7e-7; 1 / (1 + 0.3 |x|) has 3 roundings, which P passes on at most
    twofold, its eight steps count at most 10, the products 2, e 3 and x^2 / 2 times 2.5 (the roundings of its exponent): 22
    roundings and 1.25 x^2.  swish: 1 / (1 + e) takes its share (1 - s) of e's 2 |x| + 2 roundings and adds 3.
    What is kept is a code times its scale, one rounding; no slope changes faster than at 0.8."""
    def parts(v):
        if kind == "gelu":
            tail, phi = 0.5 * torch.erfc(v.abs() / math.sqrt(2)), 0.5 * torch.erfc(-v / math.sqrt(2))
            return tail * (1.7e-7 + (22 + 1.25 * v * v) * U) + 2 * U * phi, phi, torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
        s = torch.sigmoid(v)
        return s * (2 * v.abs() * (1 - s) + 5) * U, s, None

    x, kept = x.double(), kept.double()
    off, level, _ = parts(x)
    y = x.abs() * (off + U * level + 1e-37)
    off, level, density = parts(kept)
    if kind == "gelu":
        slope = off + kept.abs() * density * (7 + 1.25 * kept * kept) * U
    else:
        slope = off * (1 + kept.abs()) + 4 * U * level * (1 + kept.abs())
    return y * 1.01, (slope + 0.8 * U * kept.abs() + 1e-37) * 1.01
