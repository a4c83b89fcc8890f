"""How near the activations that keep their input come to their definitions in 64 bits: every 16-bit input, 32-bit inputs over
the whole range, and the same formulas in elementary 32-bit operations beside them.

The bounds count roundings of U = 2^-24; the hardware's exponential and reciprocal are off by one last place, 2 U.
swish: e has 2 U and a correction's rounding, 3 U, of which the sum 1 + e passes on no more; it adds U, and the quotient, which
is corrected by its residual, U: 5 U and some of the second order.  gelu, tail = e R, t = |x|: the exponent t^2 / 2 has 2.5
roundings, 1.25 t^2 U of e, and the exponential 2 U more; R = 1/2 + w Q(w) has w off by 4 U, which R passes on 0.19 / R fold (the largest of
|w R'(w)| is 0.19), and w Q(w), at most 0.47, by some 6 U: 4 U / R together, its own sum's rounding and the fit's 0.4 U; then e R,
1 - tail and the product with x: a rounding each."""
import math

import pytest
import torch

from approxtrain_amd import functors, math_ops
from tests import rows_reference as ref

pytestmark = pytest.mark.gpu

U = ref.U
KINDS = ["gelu", "swish"]


def nearest(v, dtype):
    """64-bit ``v`` rounded to the nearest number of ``dtype`` at once, ties to even."""
    bits, least = (8, -125) if dtype == torch.bfloat16 else (11, -13)
    exponent = torch.frexp(v).exponent.clamp(min=least)
    step = torch.ldexp(torch.ones_like(v), exponent - bits)
    return torch.round(v / step) * step


def bound(kind, x):
    """Of the value at x (64 bits), before it is rounded to 16 bits."""
    value = ref.ACTIVATIONS[kind][0](x).abs()
    if kind == "swish":
        return 5.2 * U * value + 2.0 ** -149
    t = x.abs()
    tail = 0.5 * torch.special.erfc(t / math.sqrt(2))
    r = 0.5 * torch.special.erfcx(t / math.sqrt(2))
    off = tail * (1.25 * t * t + 6 + 4 / r) * U
    return t * (off + U * (x > 0)) + U * value + t * 2.0 ** -126 * 1.01  # (an exponential below 2^-126 is zero)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_every_16_bit_input(dtype, kind):
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    x = x[torch.isfinite(x)]
    got = math_ops.activationi8(x.cuda()[None], kind)[0].double().cpu()
    d = x.double()
    want, off = ref.ACTIVATIONS[kind][0](d), bound(kind, d)
    low, high = nearest(want - off, dtype), nearest(want + off, dtype)
    bad = ~((got >= low) & (got <= high))
    assert not bad.any(), (x[bad][:8].tolist(), got[bad][:8].tolist(), want[bad][:8].tolist())


@pytest.mark.parametrize("kind,dtype,inputs", [
    # a last place of 32 bits from the middle of two neighbours and more, or at the lower end of the range
    ("swish", torch.bfloat16, [5.9375, -87.5, -88.0, -88.5, -89.0, -89.5, -90.0, -90.5, -91.0, -91.5]),
    ("gelu", torch.float16, [0.0003864765167236328, 0.0005464553833007812, 0.001338958740234375, 0.02783203125, -0.0003864765167236328,
                             -0.001338958740234375, -0.02783203125])], ids=["swish", "gelu"])
def test_results_beside_the_middle_of_two_neighbours(kind, dtype, inputs):
    x = torch.tensor(inputs, dtype=dtype)
    assert x.double().tolist() == inputs
    got = math_ops.activationi8(x.cuda()[None], kind)[0].double().cpu()
    assert got.tolist() == nearest(ref.ACTIVATIONS[kind][0](x.double()), dtype).tolist()


RANGES = [(-0.01, 0.01), (-1, 0), (0, 1), (-4, -1), (1, 6), (-12, -4), (-64, -12), (-87, -64), (-104, -87), (60, 70)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("low,high", RANGES)
def test_32_bit_inputs(low, high, kind):
    x = low + (high - low) * torch.rand((64, 4096), generator=torch.Generator().manual_seed(1))
    got = math_ops.activationi8(x.cuda(), kind).double().cpu()
    want, off = ref.ACTIVATIONS[kind][0](x.double()), bound(kind, x.double())
    assert ((got - want).abs() <= off * 1.01).all(), float(((got - want).abs() / off).max())


def plain(kind, x):
    if kind == "gelu":
        phi = 0.5 * torch.erfc(x * -math.sqrt(0.5))
        return x * phi, phi + x * torch.exp(x * x * -0.5) * (1 / math.sqrt(2 * math.pi))
    s = 1 / (1 + torch.exp(-x))
    return x / (1 + torch.exp(-x)), s + x * s * (1 - s)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("low,high", [(-0.01, 0.01), (-1, 0), (0, 1), (-4, -1), (1, 6), (-12, -4)])
def test_as_exact_as_elementary_32_bit_operations(low, high, kind):
    """Root mean square of what values and slopes are off by, beside the same formulas written in torch: as many roundings, so
    half as much again at most (single ones fall out one way or the other)."""
    x = (low + (high - low) * torch.rand((256, 4096), generator=torch.Generator().manual_seed(2))).cuda()
    kept = functors.keep8(x).values()
    leaf = x.clone().requires_grad_()
    y = math_ops.activationi8(leaf, kind)
    slope, = torch.autograd.grad(y, [leaf], torch.ones_like(leaf))
    value_of, slope_of = ref.ACTIVATIONS[kind]
    for got, other, want in ((y.detach(), plain(kind, x)[0], value_of(x.double())), (slope, plain(kind, kept)[1], slope_of(kept.double()))):
        off, others = ((t.double() - want).square().mean().sqrt() for t in (got, other))
        assert off <= 1.5 * others, (float(off), float(others))


@pytest.mark.parametrize("kind", KINDS)
def test_slopes_at_the_ends_of_the_range(kind):
    x = torch.tensor([-3.0e38, -1e4, -200.0, -110.0, -103.0, -95.0, -88.0, -80.0, -65.0, -64.0, -63.0, 63.0, 64.0, 65.0, 1e4, 3.0e38])[:, None]
    kept = ref.int8_values(x).float()
    leaf = x.cuda().requires_grad_()
    y = math_ops.activationi8(leaf, kind)
    slope, = torch.autograd.grad(y, [leaf], torch.ones_like(leaf))
    want = ref.ACTIVATIONS[kind][1](kept.double().clamp(-1e4, 1e4))
    assert ((slope.double().cpu() - want).abs() <= 16 * U * want.abs() + 2.0 ** -126).all()
    value = ref.ACTIVATIONS[kind][0](x.double())
    assert ((y.detach().double().cpu() - value).abs() <= 16 * U * value.abs() + 2.0 ** -120).all()
