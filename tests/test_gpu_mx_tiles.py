"""Every kind of tile, of split and of pair that the planner picks for 4-bit products, at extents that fill none of them, and
tensors whose offsets need more than 32 bits.  The plans are asserted, on the host too, so that a refit of the planner
cannot take a kernel out of these tests unseen.

Products are compared with those of the operands' own values in 64 bits: a rounding of at most 2^-23 of the running sum of
magnitudes for each block of 32, up to 16 for the sums of a split reduction, 3 for the bias and the last ones; a result
of 16 bits half a step more."""
import ctypes as C

import pytest
import torch

from approxtrain_amd import functors, load_library, math_ops

# (rows and columns of the tile, splits), m, n, k
PRODUCTS = [((256, 256, 1), 4095, 4093, 1025), ((256, 256, 1), 4001, 4003, 4000), ((256, 256, 1), 7937, 2001, 400), ((256, 256, 1), 1023, 12003, 2000),
            ((256, 256, 4), 130, 12003, 66000), ((256, 256, 1), 4095, 16381, 16400), ((256, 128, 1), 7937, 1021, 40), ((256, 128, 1), 1023, 8191, 129),
            ((256, 128, 1), 4097, 4095, 700), ((256, 128, 1), 7937, 8191, 400), ((128, 128, 1), 6001, 1021, 40), ((128, 128, 1), 130, 12003, 8200),
            ((128, 128, 4), 130, 4093, 66000), ((64, 64, 1), 1500, 2500, 300), ((64, 64, 13), 130, 131, 8200)]
# ... of the two products of a backward pass, rows, width, units
GRADIENTS = [((256, 256, 1, 1), 4095, 2001, 4093), ((256, 128, 1, 1), 1023, 4093, 1021), ((256, 128, 1, 4), 8191, 4093, 130),
             ((256, 128, 1, 8), 16383, 2047, 300), ((128, 128, 1, 1), 1023, 4093, 300), ((128, 128, 1, 4), 16383, 301, 1021),
             ((128, 128, 1, 2), 16383, 1023, 1021), ((64, 64, 1, 8), 8191, 131, 130), ((64, 64, 1, 0), 20000, 40, 33)]


def plan(*extents):
    lib = load_library()
    lib.amsim_mxfp4_plan.argtypes = [C.c_int, C.c_void_p, C.c_void_p]
    e, info = (C.c_int64 * (3 * len(extents)))(*[v for x in extents for v in x]), (C.c_int64 * 4)()
    assert lib.amsim_mxfp4_plan(len(extents), C.addressof(e), C.addressof(info)) == 0
    return tuple(info)


@pytest.mark.parametrize("want,m,n,k", PRODUCTS)
def test_plans_of_products(want, m, n, k):
    assert plan((m, n, k)) == want + (0,)


@pytest.mark.parametrize("want,m,width,units", GRADIENTS)
def test_plans_of_gradients(want, m, width, units):
    assert plan((m, width, units), (width, units, m)) == want


def test_plans_refuse():
    lib = load_library()
    lib.amsim_mxfp4_plan.argtypes = [C.c_int, C.c_void_p, C.c_void_p]
    e, info = (C.c_int64 * 6)(*[64] * 5, 0), (C.c_int64 * 4)()
    call = lib.amsim_mxfp4_plan
    assert call(0, C.addressof(e), C.addressof(info)) == call(3, C.addressof(e), C.addressof(info)) == call(1, None, C.addressof(info)) == 1
    assert call(1, C.addressof(e), None) == 1 and call(2, C.addressof(e), C.addressof(info)) == 6 and call(1, C.addressof(e), C.addressof(info)) == 0


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def assert_rows(got, a, c, bias, relu, step=2000):
    """Rows of ``got`` against those of a . c^T + bias, float64, in pieces."""
    k = a.shape[1]
    for rows in torch.arange(got.shape[0], device="cuda").split(step):
        z, size = a[rows] @ c.t(), a[rows].abs() @ c.abs().t()
        if bias is not None:
            z, size = z + bias.double(), size + bias.double().abs()
        if relu:
            z = z.clamp(min=0)
        tol = (-(-k // 32) + 19) * 2.0 ** -23 * size
        if got.dtype != torch.float32:
            info = torch.finfo(got.dtype)
            tol = tol * 1.01 + z.abs() * info.eps / 2 + info.smallest_normal * info.eps
        bad = ~((got[rows].double() - z).abs() <= tol)
        assert not bool(bad.any()), f"{int(bad.sum())} outside, the first at {[int(v[0]) for v in bad.nonzero(as_tuple=True)]} of rows from {int(rows[0])}"


@pytest.mark.gpu
@pytest.mark.parametrize("want,m,n,k", PRODUCTS)
def test_products(want, m, n, k):
    x, w, bias = (torch.randn(s, device="cuda", generator=gen(i)) for i, s in enumerate(((m, k), (n, k), (n,))))
    p, q = functors.mxfp4_quantize(x), functors.mxfp4_quantize(w)
    a, c = p.dequantize().double(), q.dequantize().double()
    assert_rows(functors.mxfp4_matmul(p, q), a, c, None, False)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = functors.mxfp4_matmul(p, q, bias, "relu", dtype)
        assert_rows(got, a, c, bias, True)
        assert torch.equal(got, functors.mxfp4_matmul(p, q, bias, "relu", dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("want,m,width,units", GRADIENTS)
def test_gradients(want, m, width, units, dtype):
    x, w, dy = (torch.randn(s, device="cuda", generator=gen(i)).to(t) for i, (s, t) in
                enumerate((((m, width), dtype), ((width, units), torch.float32), ((m, units), dtype))))
    b = torch.zeros(units, device="cuda", requires_grad=True)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = math_ops.linearmx(xl, wl, b, activation="relu")
    gx, gw, gb = torch.autograd.grad(out, [xl, wl, b], dy)
    assert (gx.dtype, gw.dtype, gb.dtype) == (dtype, torch.float32, torch.float32)
    dz = torch.where(out > 0, dy, torch.zeros_like(dy))
    (_, xc), (wr, _), (gr, gc) = (functors.mxfp4_quantize_both(t) for t in (x, w, dz))
    for got, p, q in ((gx, gr, wr), (gw, xc, gc)):
        assert_rows(got, p.dequantize().double(), q.dequantize().double(), None, False)
    # runs of up to 32 in 32 bits, those added in 16 runs of ceil(m / 512), those in order
    assert bool(((gb.double() - dz.double().sum(0)).abs() <= (32 + -(-m // 512) + 16) * 2.0 ** -24 * dz.double().abs().sum(0)).all())


@pytest.mark.gpu
def test_a_reduction_over_operands_past_32_bit_offsets():
    """More than 2^32 values in one operand: products of its rows, the last among them, are those of these rows alone.  (The
    tolerance is about 12; the reduction's last twentieth alone adds up to some 59.)"""
    rows, cols = 70001, 65536
    x = torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda").normal_(generator=gen(1))
    big, few = functors.mxfp4_quantize(x, axis=0), functors.mxfp4_quantize(x[:, :67].contiguous(), axis=0)
    got = functors.mxfp4_matmul(big, few)
    c = few.dequantize().double()
    for first in (0, 32768 - 100, cols - 300):
        part = functors.mxfp4_quantize(x[:, first:first + 300].contiguous(), axis=0)
        assert_rows(got[first:first + 300], part.dequantize().double(), c, None, False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_results_past_32_bit_offsets(dtype):
    """More than 2^31 elements of a result."""
    m, n, k = 66001, 33003, 100
    x, w = (torch.randn(s, device="cuda", generator=gen(i)) for i, s in enumerate(((m, k), (n, k))))
    p, q = functors.mxfp4_quantize(x), functors.mxfp4_quantize(w)
    got = functors.mxfp4_matmul(p, q, activation="relu", dtype=dtype)
    assert got.numel() > 1 << 31
    a, c = p.dequantize().double(), q.dequantize().double()
    middle = (1 << 31) // n
    for first in (0, middle - 300, m - 500):
        assert_rows(got[first:first + 500], a[first:first + 500], c, None, True)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_an_optimizer_s_tensor_past_32_bit_offsets(bits):
    """More than 2^31 elements, and a tensor behind them: their ends step as they do alone."""
    n, last = (1 << 31) + 70001, 5000
    params = [torch.empty(s, device="cuda", dtype=torch.bfloat16).normal_(generator=gen(i)) for i, s in enumerate((n, last))]
    grads = [torch.empty(s, device="cuda", dtype=torch.bfloat16).normal_(generator=gen(2 + i)) for i, s in enumerate((n, last))]
    pieces = [(0, 0, 5120), (0, 1 << 31, 5120), (0, n // 256 * 256 - 5120, 5120 + n % 256), (1, 0, last)]
    alone = [params[t][at:at + size].clone() for t, at, size in pieces]
    state = functors.AdamWState(params, bits)
    for step in (1, 2):
        functors.adamw_step(state, grads, step)
    for (t, at, size), p in zip(pieces, alone):
        one = functors.AdamWState([p], bits)
        for step in (1, 2):
            functors.adamw_step(one, [grads[t][at:at + size].clone()], step)
        begin = state.starts[t] + at
        assert torch.equal(params[t][at:at + size], p)
        assert torch.equal(state.m[begin:begin + one.m.numel()], one.m) and torch.equal(state.v[begin:begin + one.v.numel()], one.v)
