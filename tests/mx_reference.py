"""MXFP4 and AdamW by their definitions, in 64 bits (and, for 8-bit moments, in 32 bits step by step) on the host."""
import numpy as np

NUMBERS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def mx_values(x, axis=-1):
    """Values of x in MXFP4 with blocks of 32 along ``axis``, float64."""
    x = np.moveaxis(np.asarray(x, np.float64), axis, -1)
    n = x.shape[-1]
    pad = np.zeros(x.shape[:-1] + (-n % 32,))
    b = np.concatenate([x, pad], -1).reshape(x.shape[:-1] + (-1, 32))
    bad = ~np.isfinite(b).all(-1, keepdims=True)
    a = np.where(bad, 0.0, np.abs(b))
    _, e = np.frexp(a.max(-1, keepdims=True))
    scale = np.ldexp(1.0, np.maximum(np.where(a.max(-1, keepdims=True) > 0, e - 3, -127), -127))
    t = a / scale
    # the nearest number; of two, the one with an even code
    d = np.abs(t[..., None] - NUMBERS)
    nearest = d.min(-1, keepdims=True) == d
    q = np.where(nearest[..., 0::2].any(-1), NUMBERS[0::2][nearest[..., 0::2].argmax(-1)], NUMBERS[1::2][nearest[..., 1::2].argmax(-1)])
    v = np.where(bad, np.nan, np.copysign(q * scale, b))
    return np.moveaxis(v.reshape(x.shape[:-1] + (-1,))[..., :n], -1, axis)


def adamw(p, g, m, v, step, lr, beta1, beta2, eps, weight_decay, grad_scale=1.0):
    """(p, m, v) after a step, float64."""
    p, g, m, v = (np.asarray(t, np.float64) for t in (p, g, m, v))
    g = g * grad_scale
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    p = p * (1 - lr * weight_decay) - lr * (m / (1 - beta1 ** step)) / (np.sqrt(v / (1 - beta2 ** step)) + eps)
    return p, m, v


def decode(codes, scales, roots):
    """Moments of whole blocks of 256 from their 8-bit codes, float32."""
    c = np.asarray(codes, np.int64).reshape(-1, 256)
    bits, largest = (4, 255) if roots else (3, 127)
    mag = c if roots else c % 128
    below = largest - mag
    binade = -(-below // (1 << bits))
    f = np.where(mag > 0, np.ldexp(1.0 + (binade * (1 << bits) - below) / (1 << bits), -binade), 0.0).astype(np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        v = f * np.asarray(scales, np.float32).reshape(-1, 1)
    if not roots:
        v = np.where(c >= 128, -v, v)
    return v.reshape(-1)


def encode(x, roots):
    """Nearest 8-bit codes (ties to the even 32-bit form) and scales of float32 moments in whole blocks of 256."""
    x = np.asarray(x, np.float32).reshape(-1, 256)
    bits, largest = (4, 255) if roots else (3, 127)
    scale = np.abs(x).max(-1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        t = np.where(scale > 0, (np.abs(x) / scale).astype(np.float32), 0).astype(np.float64)
    below = largest - np.arange(1, largest + 1)
    binade = -(-below // (1 << bits))
    table = np.concatenate([[0.0], np.ldexp(1.0 + (binade * (1 << bits) - below) / (1 << bits), -binade)])
    hi = np.clip(np.searchsorted(table, t), 1, largest)
    lo = hi - 1
    up, down = table[hi] - t, t - table[lo]
    c = np.where(up < down, hi, np.where(down < up, lo, np.where(hi % 2 == 1, hi, lo)))
    # (codes are counted so that an even 32-bit form has an odd code: 1.0 is the largest, an odd one)
    if roots:
        c = np.where((t > 0) & (c == 0), 1, c)
    else:
        c = np.where(lo == 0, np.where(t < table[1] * 0.5, 0, 1), c)
        c = np.where(x < 0, c + 128, c)
    return c.astype(np.uint8).reshape(-1), scale.reshape(-1)


def adamw_8bit(p, g, codes, scales, roots, root_scales, step, lr, beta1, beta2, eps, weight_decay, grad_scale=None):
    """One step with 8-bit moments, each operation rounded to 32 bits: (p, m codes, m scales, root codes, root scales)."""
    f = np.float32
    with np.errstate(invalid="ignore", over="ignore", under="ignore"):
        p, g = np.asarray(p, f), np.asarray(g, f)
        if grad_scale is not None:
            g = g * f(grad_scale)
        m, r = decode(codes, scales, False), decode(roots, root_scales, True)
        v = r * r
        m = m * f(beta1) + g * f(1 - beta1)
        v = v * f(beta2) + (g * f(1 - beta2)) * g
        r = np.sqrt(v)
        denominator = r * f(1 / np.sqrt(1 - beta2 ** step)) + f(eps)
        p = p * f(1 - lr * weight_decay) - (m / denominator) * f(lr / (1 - beta1 ** step))
        return (p,) + encode(m, False) + encode(r, True)
