"""MXFP4 conversion, products and the layer's gradients against their definitions in 64 bits.

Values of operands are compared exactly.  A product's error: the products of elements are exact, each of the
ceil(K / 32) blocks, the bias and the sums of a split reduction add one rounding of at most 2^-23 of the running sum
of magnitudes (an instruction may cut bits instead of rounding them), and a result of 16 bits is off by half a
step more."""
import numpy as np
import pytest
import torch

from approxtrain_amd import AmsimError, functors, load_library, math_ops
from tests import mx_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def host64(t):
    return t.detach().double().cpu().numpy()


def make(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp2(torch.randint(-6, 7, (shape[-1],), generator=g).float()) * scale
    x[torch.rand(shape, generator=g) < 0.1] = 0.0
    return x.to(DTYPES[dtype])


def assert_values(q, want, dtype=torch.float32):
    got = host64(q.dequantize(dtype))
    assert got.shape == want.shape
    want = torch.from_numpy(np.ascontiguousarray(want)).to(dtype).double().numpy()
    assert np.array_equal(got, want, equal_nan=True), f"{(got != want).sum()} of {got.size} differ"


def assert_product(got, a, b, bias=None, relu=False, splits=16):
    """``got`` against relu(a . b^T + bias) of float64 operands that hold the 4-bit values."""
    z, mag = a @ b.T, np.abs(a) @ np.abs(b).T
    if bias is not None:
        z, mag = z + bias, mag + np.abs(bias)
    if relu:
        z = np.where(z < 0, 0.0, z)
    k = a.shape[1]
    tol = (-(-k // 32) + 2 + splits) * 2.0 ** -23 * mag
    if got.dtype != torch.float32:
        tol = tol * 1.01 + torch.finfo(got.dtype).eps / 2 * np.abs(z) + torch.finfo(got.dtype).tiny
    g = host64(got)
    assert g.shape == z.shape
    bad = ~(np.abs(g - z) <= tol) & ~(np.isnan(g) & np.isnan(z))
    assert not bad.any(), f"{bad.sum()} of {bad.size} outside; worst {np.nanmax(np.abs(g - z) / np.maximum(tol, 1e-300)):.3g} of the tolerance"


SHAPES = [(1, 1), (1, 31), (1, 32), (1, 33), (2, 64), (15, 128), (16, 129), (17, 127), (33, 31), (64, 128), (65, 260), (128, 128),
          (130, 257), (300, 77), (1, 4096), (517, 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values_of_rows_columns_and_both(shape, dtype):
    x = make(shape, dtype, 1)
    rows, cols = ref.mx_values(host64(x), 1), ref.mx_values(host64(x), 0).T
    d = x.cuda()
    assert_values(functors.mxfp4_quantize(d), rows)
    assert_values(functors.mxfp4_quantize(d, axis=0), cols)
    r, c = functors.mxfp4_quantize_both(d)
    assert_values(r, rows, DTYPES[dtype])
    assert_values(c, cols, DTYPES[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_of_special_blocks(dtype):
    t = DTYPES[dtype]
    info = torch.finfo(t)
    x = torch.zeros(64, 128)
    grid = torch.tensor([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, 7.5, 7.75])
    x[0, :18], x[1, :18], x[2, :18] = grid, -grid, grid * 2.0 ** -9
    x[3, 5], x[4, 40], x[5, 70], x[6, :] = float("inf"), float("-inf"), float("nan"), float("nan")
    x[7, :], x[8, 3], x[9, 3] = info.max, info.max, -info.max
    x[10, :4] = torch.tensor([info.tiny, info.tiny / 2, -info.tiny / 4, info.tiny * info.eps])
    x[11, :33] = info.tiny * info.eps                                     # the smallest subnormal
    x[12, :64] = -0.0
    x[13, :] = torch.linspace(-8, 8, 128)
    x = x.to(t)
    d = x.cuda()
    assert_values(functors.mxfp4_quantize(d), ref.mx_values(host64(x), 1))
    assert_values(functors.mxfp4_quantize(d.t().contiguous(), axis=0), ref.mx_values(host64(x), 1))
    assert_values(functors.mxfp4_quantize_both(d)[1], ref.mx_values(host64(x), 0).T)
    # signs of zeros
    got = functors.mxfp4_dequantize(functors.mxfp4_quantize(d))[12].cpu()
    assert torch.equal(torch.signbit(got), torch.signbit(x[12].float()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
    base = make((70, 300), dtype, 2).cuda()
    views = {"slice": base[3:60, 16:272], "odd start": base[1:, 1:140], "transposed": base.t(), "transposed slice": base[:41, 5:].t(),
             "stepped": base[::2, ::3], "expanded": base[:1].expand(40, 300), "one row": base[5:6, 7:90], "one column": base[:, 9:10]}
    for name, v in views.items():
        want = host64(v)
        r, c = functors.mxfp4_quantize_both(v)
        assert_values(r, ref.mx_values(want, 1)), name
        assert_values(c, ref.mx_values(want, 0).T), name
        assert_values(functors.mxfp4_quantize(v, axis=-2), ref.mx_values(want, 0).T), name


PRODUCTS = [(1, 1, 1), (1, 17, 33), (5, 3, 128), (16, 16, 128), (17, 65, 129), (64, 64, 256), (100, 130, 260), (128, 300, 784), (33, 1, 1000),
            (257, 255, 96), (300, 515, 130), (31, 33, 9000), (512, 512, 640), (1030, 700, 384)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_products(m, n, k):
    x, w = make((m, k), "f32", 3), make((n, k), "f32", 4)
    a, b = functors.mxfp4_quantize(x.cuda()), functors.mxfp4_quantize(w.cuda())
    va, vb = ref.mx_values(host64(x)), ref.mx_values(host64(w))
    assert_product(functors.mxfp4_matmul(a, b), va, vb)
    for i, (name, t) in enumerate(DTYPES.items()):
        bias = make((1, n), name, 5 + i)[0]
        got = functors.mxfp4_matmul(a, b, bias.cuda(), "relu", t)
        assert got.dtype == t
        if name == "f16":
            assert_product(got, va, vb, host64(bias), True) if np.abs(va @ vb.T).max() < 6e4 else None
        else:
            assert_product(got, va, vb, host64(bias), True)


def test_random_products():
    r = np.random.default_rng(11)
    for case in range(40):
        m, n, k = (int(np.exp(r.uniform(0, np.log(hi)))) for hi in (700, 700, 1500))
        x, w = make((m, k), "bf16", 100 + case), make((k, n), "bf16", 200 + case)
        got = functors.mxfp4_matmul(functors.mxfp4_quantize(x.cuda()), functors.mxfp4_quantize(w.cuda(), axis=0))
        assert_product(got, ref.mx_values(host64(x)), ref.mx_values(host64(w), 0).T)


def test_products_run_to_run_and_on_another_stream():
    a, b = (functors.mxfp4_quantize(make((n, 3000), "f32", n).cuda()) for n in (60, 90))
    want = functors.mxfp4_matmul(a, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = functors.mxfp4_matmul(a, b)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(want, again) and torch.equal(want, functors.mxfp4_matmul(a, b))


def test_a_block_that_is_not_finite_reaches_its_own_rows_only():
    x, w = make((40, 500), "f32", 6), make((50, 500), "f32", 7)
    x[3, 100], w[7, 499] = float("inf"), float("nan")
    got = functors.mxfp4_matmul(functors.mxfp4_quantize(x.cuda()), functors.mxfp4_quantize(w.cuda()), activation="relu").cpu()
    bad = torch.zeros(40, 50, dtype=torch.bool)
    bad[3], bad[:, 7] = True, True
    assert torch.equal(torch.isnan(got), bad)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 10, 33), (1, 4096, 4096), (2, 100, 784), (7, 333, 130), (13, 1003, 2051), (16, 64, 128), (17, 64, 128), (40, 90, 1100),
                                   (200, 70, 300)])
def test_linear_of_raw_activations(m, n, k, dtype):
    """The fused form quantises its activations as the conversion does, and one row of many like one row alone."""
    x, w, bias = make((m, k), dtype, 8, 0.1), make((k, n), dtype, 9, 0.1), make((1, n), "f32", 10)[0]
    weights = functors.mxfp4_quantize(w.cuda(), axis=0)
    got = functors.mxfp4_linear(x.cuda(), weights, bias.cuda(), "relu")
    assert got.dtype == x.dtype
    assert_product(got, ref.mx_values(host64(x)), ref.mx_values(host64(w), 0).T, host64(bias), True)
    wide = torch.zeros(m, k + 3, dtype=x.dtype, device="cuda")
    wide[:, 1:k + 1] = x.cuda()
    assert torch.equal(functors.mxfp4_linear(wide[:, 1:k + 1], weights, bias.cuda(), "relu"), got)
    x[0, k // 2] = float("nan")
    bad = torch.isnan(functors.mxfp4_linear(x.cuda(), weights)).cpu()
    assert bad[0].all() and not bad[1:].any()


def test_linear_of_leading_axes():
    x, w = make((24, 96), "bf16", 12).cuda(), make((96, 40), "bf16", 13).cuda()
    weights = functors.mxfp4_quantize(w, axis=0)
    want = functors.mxfp4_linear(x, weights)
    assert torch.equal(functors.mxfp4_linear(x.reshape(2, 3, 4, 96), weights), want.reshape(2, 3, 4, 40))
    assert torch.equal(functors.mxfp4_linear(x[0], weights), functors.mxfp4_linear(x[:1], weights)[0])
    assert functors.mxfp4_linear(x.reshape(2, 12, 96)[:, :0], weights).shape == (2, 0, 40)
    assert torch.equal(functors.mxfp4_linear(x.t().contiguous().t(), weights), want)


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("m,width,units,dtype,kernel_dtype", [(1, 40, 10, "f32", "f32"), (128, 784, 300, "f32", "f32"), (70, 130, 33, "bf16", "f32"),
                                                              (33, 64, 257, "f16", "f16"), (300, 96, 1, "bf16", "bf16"), (2050, 70, 40, "f32", "f32")])
def test_gradients_against_the_formula(m, width, units, dtype, kernel_dtype, relu):
    x, w, b = make((m, width), dtype, 20, 0.1), make((width, units), kernel_dtype, 21, 0.1), make((1, units), "f32", 22)[0]
    dy = make((m, units), dtype, 23, 0.01)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    out = math_ops.linearmx(*leaves, activation="relu" if relu else None)
    gx, gw, gb = torch.autograd.grad(out, leaves, dy.cuda())
    assert (gx.dtype, gw.dtype, gb.dtype) == (x.dtype, w.dtype, b.dtype)
    assert_product(out, ref.mx_values(host64(x)), ref.mx_values(host64(w), 0).T, host64(b), relu)
    dz = host64(dy) * ((host64(out) > 0) if relu else 1.0)
    assert_product(gx, ref.mx_values(dz), ref.mx_values(host64(w)))
    assert_product(gw, ref.mx_values(host64(x), 0).T, ref.mx_values(dz, 0).T)
    # 32-bit sums of m terms
    assert (np.abs(host64(gb) - dz.sum(0)) <= (m + 1) * 2.0 ** -24 * np.abs(dz).sum(0)).all()


def test_gradients_against_differences():
    """On the format's own numbers, at steps that stay on them, the layer is linear in each operand: differences
    of its outputs are its gradients without error."""
    r = np.random.default_rng(5)
    x = torch.from_numpy(r.choice([-1.0, 0.0, 1.0], (6, 64))).float()
    w = torch.from_numpy(r.choice([-1.0, 0.0, 1.0], (64, 33))).float()
    x[:, ::32], x[0], w[::32] = 4.0, 4.0, 4.0     # every block's scale is 1, along either axis
    w[:, 0], w[:, 32] = 4.0, 4.0
    b = torch.zeros(33)
    dy = torch.from_numpy(r.choice([-1.0, 0.5, 2.0], (6, 33))).float()
    dy[0], dy[:, ::32] = 4.0, 4.0
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(math_ops.linearmx(*leaves), leaves, dy.cuda())

    def loss(*tensors):
        return float((math_ops.linearmx(*[t.cuda() for t in tensors]).double() * dy.cuda().double()).sum())

    for which, (i, j) in ((0, (2, 5)), (0, (5, 63)), (1, (7, 3)), (1, (40, 20)), (2, (4, 0))):
        moved = [t.clone() for t in (x, w, b)]
        at = moved[which][i] if which == 2 else moved[which][i, j]
        before = float(at)
        if which == 2:
            moved[2][i] = before + 0.5
        else:
            moved[which][i, j] = before + 0.5
        got = grads[which][i] if which == 2 else grads[which][i, j]
        assert (loss(*moved) - loss(x, w, b)) / 0.5 == float(got), (which, i, j)


def test_gradients_of_a_view_of_few_and_of_no_wanted_operands():
    x, w = make((2, 9, 50), "f32", 30).cuda(), make((50, 21), "f32", 31).cuda()
    y = math_ops.linearmx(x, w)
    assert y.shape == (2, 9, 21) and not y.requires_grad
    wg = w.clone().requires_grad_()
    gw, = torch.autograd.grad(math_ops.linearmx(x, wg).sum(), [wg])           # (a gradient of stride 0)
    assert_product(gw, ref.mx_values(host64(x.reshape(18, 50)), 0).T, ref.mx_values(np.ones((18, 21)), 0).T)
    xg = x.clone().requires_grad_()
    gx, = torch.autograd.grad(math_ops.linearmx(xg, w).transpose(0, 1).sum(), [xg])
    assert_product(gx.reshape(18, 50), ref.mx_values(np.ones((18, 21))), ref.mx_values(host64(w)))
    b = torch.zeros(21, device="cuda", requires_grad=True)
    gb, = torch.autograd.grad(math_ops.linearmx(x, w, b).sum(), [b])
    assert torch.equal(gb, torch.full((21,), 18.0, device="cuda"))
    with torch.no_grad():
        assert torch.equal(math_ops.linearmx(xg, wg), y)


def test_training_step_in_a_graph():
    """Forward and backward captured once; every replay, with eager work between, against the eager result."""
    x, w, b = make((200, 130), "bf16", 40).cuda(), make((130, 70), "f32", 41, 0.1).cuda(), make((1, 70), "f32", 42)[0].cuda()
    dy = make((200, 70), "bf16", 43).cuda()
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]

    def step(leaves):
        out = math_ops.linearmx(*leaves, activation="relu")
        return (out.detach(),) + torch.autograd.grad(out, leaves, dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(leaves)
    for seed in (1, 2, 3):
        new = [make((200, 130), "bf16", 50 + seed).cuda(), make((130, 70), "f32", 60 + seed, 0.1).cuda(), make((1, 70), "f32", 70 + seed)[0].cuda()]
        with torch.no_grad():
            for leaf, v in zip(leaves, new):
                leaf.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        want = step([v.requires_grad_() for v in new])
        for g, e in zip(captured, want):
            assert torch.equal(g, e)


@pytest.mark.parametrize("dtype", DTYPES)
def test_tensors_larger_than_the_cache(dtype):
    """More than 224 MB: every value as pieces of the tensor convert alone."""
    rows, cols = (1900 if dtype == "f32" else 3800), 32003
    x = torch.empty((rows, cols), dtype=DTYPES[dtype], device="cuda")
    x.normal_(generator=torch.Generator(device="cuda").manual_seed(3))
    q = functors.mxfp4_quantize(x)
    r, c = functors.mxfp4_quantize_both(x)
    got, both, columns = q.dequantize(x.dtype), r.dequantize(x.dtype), c.dequantize(x.dtype)
    assert torch.equal(got, both)
    for first in range(0, rows, 600):
        assert torch.equal(got[first:first + 600], functors.mxfp4_quantize(x[first:first + 600]).dequantize(x.dtype))
    for first in range(0, cols, 8000):
        assert torch.equal(columns[first:first + 8000], functors.mxfp4_quantize(x[:, first:first + 8000], axis=0).dequantize(x.dtype))


def test_operands_past_32_bit_offsets():
    """More than 2^32 values in one tensor: its last rows and columns convert as they do alone."""
    rows, cols = 70001, 65536
    x = torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda")
    x.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    r, c = functors.mxfp4_quantize_both(x)
    tail = x[rows - 113:].clone()  # from row 69888 = 546 * 128 on
    want = functors.mxfp4_quantize(tail)
    n = want.data.numel() * 8 // 17 // 1024 * 1024
    steps = cols // 128
    assert (rows - 113) % 128 == 0
    first = (rows - 113) // 16 * steps * 1024
    codes = -(-113 // 16) * steps * 1024
    assert torch.equal(r.data[first:first + codes], want.data[:codes])
    del n
    probe = functors.mxfp4_matmul(c, functors.mxfp4_quantize_both(x[:, :3].contiguous())[1])
    assert probe.shape == (cols, 3)
    few = functors.mxfp4_matmul(functors.mxfp4_quantize(x[:, cols - 64:].contiguous(), axis=0), functors.mxfp4_quantize(x[:, :3].contiguous(), axis=0))
    mag = float(x[:, :3].float().abs().sum()) * 6
    assert float((probe[cols - 64:] - few).abs().max()) <= (rows / 32 + 20) * 2.0 ** -23 * mag


def test_refusals_with_tensors_on_the_device():
    x = torch.randn(8, 40, device="cuda")
    q, p = functors.mxfp4_quantize(x), functors.mxfp4_quantize(torch.randn(8, 41, device="cuda"))
    with pytest.raises(ValueError, match="lengths"):
        functors.mxfp4_matmul(q, p)
    with pytest.raises(ValueError, match="activation"):
        functors.mxfp4_matmul(q, q, activation="gelu")
    with pytest.raises(ValueError, match="bias"):
        functors.mxfp4_matmul(q, q, bias=torch.zeros(7, device="cuda"))
    with pytest.raises(TypeError, match="bias"):
        functors.mxfp4_matmul(q, q, bias=torch.zeros(8, device="cuda", dtype=torch.float64))
    with pytest.raises(TypeError, match="result"):
        functors.mxfp4_matmul(q, q, dtype=torch.float64)
    with pytest.raises(TypeError, match="MXTensor"):
        functors.mxfp4_matmul(x, q)
    with pytest.raises(TypeError, match="float32"):
        functors.mxfp4_quantize(x.double())
    with pytest.raises(ValueError, match="matrix"):
        functors.mxfp4_quantize(x[0])
    with pytest.raises(ValueError, match="empty"):
        functors.mxfp4_quantize(x[:0])
    with pytest.raises(ValueError, match="axis"):
        functors.mxfp4_quantize(x, axis=2)
    with pytest.raises(ValueError, match="length"):
        functors.mxfp4_linear(x, p)
    with pytest.raises(ValueError, match="linearmx"):
        math_ops.linearmx(x, torch.randn(41, 3, device="cuda"))
    out = torch.empty(8, 8, device="cuda")
    long = functors.mxfp4_quantize(torch.randn(8, 40000, device="cuda"))
    lib = load_library()
    need = lib.amsim_mxfp4_matmul_workspace_bytes(8, 8, 40000)
    if need:
        assert lib.amsim_mxfp4_matmul(long.data.data_ptr(), long.data.data_ptr(), 8, 8, 40000, None, 0, 0, out.data_ptr(), 0, None, 0, None) == 5
    with pytest.raises(AmsimError):
        functors.check(lib.amsim_mxfp4_matmul(q.data.data_ptr(), q.data.data_ptr() + 8, 8, 8, 40, None, 0, 0, out.data_ptr(), 0, None, 0, None))
