"""Products in 8-bit integers, their operands and a layer's gradients against the definitions in 64 bits.

Values of operands are compared exactly (a code times its scale, rounded once).  A product's sum is exact; it is rounded to
32 bits, multiplied by two scales and added to a bias, four roundings, and a result of 16 bits is off by half a step more."""
import ctypes as C

import pytest
import torch

from approxtrain_amd import AmsimError, functors, layers, load_library, math_ops
from tests import rows_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def make(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp2(torch.randint(-3, 4, (shape[-1],), generator=g).float()) * scale
    x[torch.rand(shape, generator=g) < 0.1] = 0.0
    return x.to(DTYPES[dtype])


def plan(*extents):
    info = (C.c_int64 * 4)()
    flat = (C.c_int64 * (3 * len(extents)))(*[v for e in extents for v in e])
    lib = load_library()
    lib.amsim_i8_plan.argtypes = [C.c_int, C.c_void_p, C.c_void_p]
    assert lib.amsim_i8_plan(len(extents), flat, info) == 0
    return list(info)


def close(got, product, bias=None, relu=False, name="out"):
    """``got`` against relu(product + bias), the product exact."""
    z = product if bias is None else product + bias.double()
    tol = 3 * ref.U * product.abs() + ref.U * z.abs()
    if relu:
        z = z.clamp(min=0)
    half = ref.half_step(got.dtype)
    tol = tol * 1.01 + (half * z.abs() * 1.01 if got.dtype != torch.float32 else 0) + torch.finfo(got.dtype).smallest_normal * half * 2
    got = got.detach().double().cpu()
    assert got.shape == z.shape, name
    bad = ~((got - z).abs() <= tol) & ~(torch.isnan(got) & torch.isnan(z))
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} outside; worst {float(((got - z).abs() / tol).nan_to_num().max()):.3g} of the tolerance"


def matmul64(a, b):
    """a . b^T of whole numbers in 64 bits (on the device for large ones: exact there as well)."""
    return (a.cuda() @ b.cuda().t().contiguous()).cpu() if a.numel() + b.numel() > 1 << 18 else a @ b.t()


SHAPES = [(1, 1), (1, 15), (1, 16), (1, 64), (2, 65), (15, 63), (16, 64), (17, 100), (33, 31), (64, 128), (65, 260), (48, 513), (130, 257), (300, 77), (1, 4096),
          (517, 1), (40, 4097), (20, 9000), (5, 20000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values_of_rows_and_columns(shape, dtype):
    x = make(shape, dtype, 1)
    x[0] *= 1e-3
    for axis, t in ((-1, x), (0, x.t())):
        q = functors.int8_quantize(x.cuda(), axis)
        assert q.shape == t.shape
        assert torch.equal(q.dequantize().cpu(), ref.int8_values(t).float())
        assert torch.equal(q.dequantize(DTYPES[dtype]).cpu(), ref.int8_values(t).float().to(DTYPES[dtype]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_operands_of_strided_matrices(dtype):
    base = make((200, 300), dtype, 2).cuda()
    for view in (base[:, 3:250], base[::2, 5:], base.t(), base[3:100].t(), base[:, ::3], base[:1].expand(20, 300), base[::-1] if False else base.flip(0)):
        for axis in (-1, 0):
            a, b = functors.int8_quantize(view, axis), functors.int8_quantize(view.contiguous(), axis)
            assert torch.equal(a.data, b.data)


def test_every_byte_of_an_operand_is_written():
    for shape in ((1, 1), (17, 70), (33, 130), (70, 17)):
        x = make(shape, "f32", 3).cuda()
        for axis in (-1, 0):
            torch.empty(1 << 20, dtype=torch.uint8, device="cuda").fill_(0xa5)
            a = functors.int8_quantize(x, axis).data.clone()
            torch.empty(1 << 20, dtype=torch.uint8, device="cuda").fill_(0x5a)
            assert torch.equal(a, functors.int8_quantize(x, axis).data)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_rows_that_are_not_finite(bad):
    x = make((70, 200), "f32", 4)
    x[37, 111] = bad
    assert torch.isnan(functors.int8_quantize(x.cuda()).dequantize()[37]).all()
    assert torch.isnan(functors.int8_quantize(x.cuda(), 0).dequantize()[111]).all()
    w = functors.int8_quantize(make((200, 30), "f32", 5).cuda(), 0)
    for rows in (slice(37, 38), slice(0, 70)):  # (one of few rows, and of many)
        out = functors.int8_linear(x[rows].cuda(), w)
        nan = torch.isnan(out).all(1)
        assert nan.sum() == 1 and torch.isfinite(out[~nan]).all()


def test_largest_and_smallest_scales():
    a = torch.tensor([[3.0e38, 1.0], [1e-30, 1e-31], [2.0 ** -125, 0.0], [0.0, 0.0]]).cuda()
    b = torch.tensor([[1e-30, 3e-31], [1e30, 1e28], [0.0, 0.0]]).cuda()
    got = functors.int8_matmul(functors.int8_quantize(a), functors.int8_quantize(b))
    (qa, sa), (qb, sb) = ref.int8(a.cpu()), ref.int8(b.cpu())
    want = (qa @ qb.t()) * sa * sb.t()
    assert want[0, 1] > 3.5e38 and torch.isinf(got[0, 1])
    want[0, 1] = 0
    got[0, 1] = 0
    close(got, want)


@pytest.mark.parametrize("m,n", [(40, 33), (200, 150), (600, 1300)])
def test_scales_of_every_size_beside_each_other(m, n):
    """Rows and columns from 1e-36 to 1e36: each result is its own definition's, and the same with whatever stands beside it."""
    x, w = make((m, 96), "f32", 1), make((n, 96), "f32", 2)
    x *= 10.0 ** torch.randint(-18, 19, (m, 1), generator=torch.Generator().manual_seed(3)).float()
    w *= 10.0 ** torch.randint(-18, 19, (n, 1), generator=torch.Generator().manual_seed(4)).float()
    x[::7] *= 1e18
    x[3::7] *= 1e-18
    a, b = functors.int8_quantize(x.cuda()), functors.int8_quantize(w.cuda())
    (qa, sa), (qb, sb) = ref.int8(x), ref.int8(w)
    want = (qa @ qb.t()) * sa * sb.t()
    assert (sa < 1e-34).any() and (sa > 1e30).any()
    got = functors.int8_matmul(a, b)
    # (from 2^128 on no numbers of 32 bits; four roundings below it either may come out)
    beyond, at_most = want.abs() >= 2.0 ** 128 * (1 + 4 * ref.U), want.abs() >= 2.0 ** 128 * (1 - 4 * ref.U)
    assert torch.isinf(got.cpu()[beyond]).all()
    close(torch.where(at_most.cuda(), 0.0, got), torch.where(at_most, 0.0, want))
    for row in (0, 3, 5, m - 1):
        assert torch.equal(functors.int8_matmul(functors.int8_quantize(x[row:row + 1].cuda()), b)[0], got[row])
    calm = (sb[:, 0] > 2.0 ** -50) & (sb[:, 0] < 2.0 ** 50)
    few = functors.int8_quantize(w[calm].cuda())
    assert torch.equal(functors.int8_matmul(a, few), got[:, calm.cuda()])


PRODUCTS = [(1, 1, 1), (1, 4096, 64), (1, 10, 70), (2, 33, 9000), (3, 1000, 4096), (5, 17, 6000), (8, 130, 4096), (9, 257, 3600), (13, 1003, 2051), (16, 64, 16384),
            (17, 100, 16384), (31, 77, 1000), (33, 200, 990), (48, 513, 640), (64, 40, 512), (64, 300, 4000), (65, 64, 64), (64, 10, 16385), (64, 8192, 192), (64, 8193, 192), (5, 8200, 1100), (100, 10, 40000),
            (129, 300, 784), (257, 515, 129), (1000, 1003, 333), (2048, 2048, 200), (300, 5000, 70), (4099, 17, 260)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", PRODUCTS, ids=str)
def test_linear_and_matmul(m, n, k, dtype):
    x, kernel, bias = make((m, k), dtype, 1), make((k, n), dtype, 2), make((n,), "f32", 3, 5.0)
    (qx, sx), (qw, sw) = ref.int8(x), ref.int8(kernel, 0)
    product = matmul64(qx, qw.t()) * sx * sw
    w = functors.int8_quantize(kernel.cuda(), 0)
    out = functors.int8_linear(x.cuda(), w, bias.cuda(), "relu")
    assert out.dtype == x.dtype
    close(out, product, bias, relu=True)
    close(functors.int8_linear(x.cuda(), w), product)
    q = functors.int8_quantize(x.cuda())
    assert torch.equal(functors.int8_matmul(q, w, bias.cuda(), "relu", x.dtype), out)
    close(functors.int8_matmul(q, w, bias.to(DTYPES[dtype]).cuda()), product, bias.to(DTYPES[dtype]))


@pytest.mark.parametrize("extents,want", [
    ((2048, 2048, 512), None), ((4096, 4096, 256), None), ((1024, 1024, 4096), None), ((200, 200, 60000), None), ((70, 60, 30000), None), ((8192, 512, 512), None),
    ((5000, 3000, 200), None), ((512, 512, 8192), None), ((100, 100, 300000), None), ((3, 40, 200000), None)])
def test_products_of_every_tile(extents, want):
    m, n, k = extents
    x, w = make((m, k), "bf16", 1).cuda(), make((n, k), "bf16", 2).cuda()
    a, b = functors.int8_quantize(x), functors.int8_quantize(w)
    info = plan((m, n, k))
    if k > 131072:
        assert info[2] >= 2  # (a sum of 32 bits has at most 131072 terms)
    (qa, sa), (qb, sb) = ref.int8(x), ref.int8(w)
    want = ((qa @ qb.t().contiguous()) * sa * sb.t()).cpu()
    for t in DTYPES.values():
        close(functors.int8_matmul(a, b, dtype=t), want, name=f"{info} {t}")


def test_the_plans_above_reach_every_tile_and_splits():
    every = [plan(e) for e in ((4096, 4096, 256), (1024, 1024, 4096), (200, 200, 60000), (8192, 512, 512), (5000, 3000, 200), (2048, 2048, 512), (512, 512, 8192))]
    assert {tuple(p[:2]) for p in every} == {(256, 256), (256, 128), (128, 128), (64, 64)}
    assert any(p[2] > 1 for p in every) and any(p[2] == 1 for p in every)
    assert plan((64, 5000, 16384))[2] == 0 and plan((65, 5000, 16384))[2] > 0


def test_the_longest_sums_do_not_wrap():
    for k in (131072, 131073, 1 << 19, 1 << 21):  # every code 127, every sum the largest there is
        x = torch.ones(2, k, device="cuda")
        got = functors.int8_matmul(functors.int8_quantize(x), functors.int8_quantize(x))
        (q, s) = ref.int8(x[:1].cpu())
        want = float((q @ q.t()).item()) * s.item() ** 2
        assert ((got.double() - want).abs() <= 4 * ref.U * want).all()


def train(x, kernel, bias, dy, relu=False):
    leaves = [t.detach().cuda().requires_grad_() for t in (x, kernel, bias)]
    out = math_ops.lineari8(*leaves, activation="relu" if relu else None)
    return out, torch.autograd.grad(out, leaves, dy.cuda())


def check_train(x, kernel, bias, dy, relu=False):
    out, (dx, dw, db) = train(x, kernel, bias, dy, relu)
    (qx, sx), (qw, sw) = ref.int8(x), ref.int8(kernel, 0)
    close(out, matmul64(qx, qw.t()) * sx * sw, bias, relu)
    g = dy.double()
    if relu:
        g = torch.where(out.detach().double().cpu() > 0, g, 0.0)
    qv, sv = ref.int8((g * sw).float())
    qu, su = ref.int8((g * sx).float(), 0)
    assert (dx.dtype, dw.dtype, db.dtype) == (x.dtype, kernel.dtype, bias.dtype)
    close(dx, matmul64(qv, qw) * sv, name="dx")
    close(dw, matmul64(qx.t(), qu.t()) * su, name="dw")
    tol = (x.shape[0] / 64 + 100) * ref.U * g.abs().sum(0) + ref.half_step(db.dtype) * g.sum(0).abs() * 1.01
    assert ((db.double().cpu() - g.sum(0)).abs() <= tol).all()
    return out, dx, dw, db


TRAINS = [(1, 1, 1), (1, 300, 70), (2, 16, 16), (16, 64, 64), (17, 65, 33), (64, 10, 1000), (65, 33, 200), (128, 300, 784), (100, 1003, 333), (513, 70, 129), (2000, 40, 50),
          (300, 2000, 100), (90, 5000, 40), (1030, 515, 260), (4100, 130, 200)]


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", TRAINS, ids=str)
def test_training_step(m, n, k, dtype, relu):
    check_train(make((m, k), dtype, 1), make((k, n), "f32", 2, 0.1), make((n,), "f32", 3), make((m, n), dtype, 4, 0.01), relu)


@pytest.mark.parametrize("kernel_dtype", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_training_step_of_every_pair_of_types(dtype, kernel_dtype):
    check_train(make((130, 200), dtype, 1), make((200, 90), kernel_dtype, 2), make((90,), kernel_dtype, 3), make((130, 90), dtype, 4))


def test_training_step_in_large_tiles():
    check_train(make((2100, 1100), "bf16", 1), make((1100, 1300), "f32", 2, 0.1), make((1300,), "f32", 3), make((2100, 1300), "bf16", 4, 0.01))


def test_training_step_of_more_tokens_than_one_sum_has():
    m, n, k = 150000, 33, 40
    assert plan((k, n, m))[2] >= 2
    check_train(make((m, k), "bf16", 1), make((k, n), "f32", 2, 0.1), make((n,), "f32", 3), make((m, n), "bf16", 4, 0.01))


def test_what_comes_back_in_another_form_is_refused():
    x, kernel = make((40, 60), "f32", 1).cuda().requires_grad_(), make((60, 30), "f32", 2).cuda().requires_grad_()
    for other in (lambda t: t[:-1], lambda t: t.cpu(), lambda t: t.view(torch.int8)):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, other):
            out = math_ops.lineari8(x, kernel)
        with pytest.raises(RuntimeError, match="in another form"):
            out.sum().backward()


def test_asked_for_some_gradients():
    x, kernel, bias, dy = make((150, 200), "bf16", 1).cuda(), make((200, 90), "f32", 2).cuda(), make((90,), "f32", 3).cuda(), make((150, 90), "bf16", 4).cuda()
    _, want = train(x, kernel, bias, dy)
    for which in range(1, 8):
        leaves = [t.clone().requires_grad_(bool(which >> i & 1)) for i, t in enumerate((x, kernel, bias))]
        got = iter(torch.autograd.grad(math_ops.lineari8(*leaves), [t for t in leaves if t.requires_grad], dy))
        for i in range(3):
            if which >> i & 1:
                g = next(got)
                if i < 2:
                    assert torch.equal(g, want[i])
                else:  # (summed in another order where x's gradient is not wanted)
                    torch.testing.assert_close(g, want[i], rtol=0, atol=float(150 * ref.U * dy.double().abs().sum(0).max()))
    leaves = [t.clone().requires_grad_() for t in (x, kernel, bias)]
    for i in range(2):
        assert torch.equal(torch.autograd.grad(math_ops.lineari8(*leaves), [leaves[i]], dy)[0], want[i])


def test_strided_and_higher_rank_inputs():
    base = make((48, 700), "f16", 1).cuda()
    kernel, bias = make((600, 70), "f32", 2, 0.1).cuda(), make((70,), "f32", 3).cuda()
    w = functors.int8_quantize(kernel, 0)
    for view in (base[:, 100:], base[::3, 50:650], make((600, 48), "f16", 2).cuda().t(), base[:, 100:].reshape(4, 12, 600), base[:1, 3:603].expand(70, 600)):
        flat = view.contiguous().reshape(-1, 600)
        want = functors.int8_linear(flat, w, bias)
        assert torch.equal(functors.int8_linear(view, w, bias), want.reshape(view.shape[:-1] + (70,)))
        a, b = view.detach().requires_grad_(), flat.clone().requires_grad_()
        dy = make((flat.shape[0], 70), "f16", 5).cuda()
        k1, k2 = kernel.t().contiguous().t().requires_grad_(), kernel.clone().requires_grad_()
        ga = torch.autograd.grad(math_ops.lineari8(a, k1, bias), [a, k1], dy.t().contiguous().t().reshape(view.shape[:-1] + (70,)))
        gb = torch.autograd.grad(math_ops.lineari8(b, k2, bias), [b, k2], dy)
        assert torch.equal(ga[0].reshape(-1, 600), gb[0]) and torch.equal(ga[1], gb[1])
    one = base[0, :600]
    assert torch.equal(functors.int8_linear(one, w), functors.int8_linear(one[None], w)[0])


def test_batches_of_no_rows():
    kernel, bias = make((20, 7), "f32", 1).cuda().requires_grad_(), torch.zeros(7, device="cuda", requires_grad=True)
    x = torch.empty(0, 20, device="cuda", requires_grad=True)
    out = math_ops.lineari8(x, kernel, bias, "relu")
    gx, gk, gb = torch.autograd.grad(out, [x, kernel, bias], torch.empty(0, 7, device="cuda"))
    assert out.shape == (0, 7) and gx.shape == (0, 20) and torch.equal(gk, torch.zeros_like(kernel)) and torch.equal(gb, torch.zeros_like(bias))
    w = functors.int8_quantize(kernel.detach(), 0)
    assert functors.int8_linear(torch.empty(3, 0, 20, device="cuda"), w).shape == (3, 0, 7)
    with torch.no_grad():
        assert math_ops.lineari8(torch.empty(2, 0, 20, device="cuda"), kernel).shape == (2, 0, 7)


def test_a_gradient_with_a_token_that_is_not_finite():
    x, kernel, bias, dy = make((80, 60), "f32", 1), make((60, 50), "f32", 2), make((50,), "f32", 3), make((80, 50), "f32", 4)
    dy[11, 7] = float("inf")
    _, (dx, dw, db) = train(x, kernel, bias, dy)
    rest = [i for i in range(80) if i != 11]
    assert torch.isnan(dx[11]).all() and torch.isfinite(dx[rest]).all()
    cols = [i for i in range(50) if i != 7]
    assert torch.isnan(dw[:, 7]).all() and torch.isfinite(dw[:, cols]).all() and torch.isinf(db[7])


def test_captured_training_steps():
    kernel, bias = make((200, 90), "f32", 2, 0.1).cuda().requires_grad_(), make((90,), "f32", 3).cuda().requires_grad_()
    xs, dy = [make((150, 200), "f32", s).cuda() for s in range(4)], make((150, 90), "f32", 9).cuda()
    leaf = xs[0].clone().requires_grad_()

    def step():
        out = math_ops.lineari8(leaf, kernel, bias, "relu")
        return (out.detach(), *torch.autograd.grad(out, [leaf, kernel, bias], dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for x in xs * 2:
        with torch.no_grad():
            leaf.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_two_graphs_and_an_eager_call_at_once():
    w = functors.int8_quantize(make((800, 300), "bf16", 1).cuda(), 0)
    xs = [make((500, 800), "bf16", s).cuda() for s in range(2)]
    want = [functors.int8_linear(x, w) for x in xs]
    graphs, outs = [], []
    for x in xs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(functors.int8_linear(x, w))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        eager = functors.int8_linear(xs[0], w)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0]) and all(torch.equal(a, b) for a, b in zip(outs, want))


def test_a_backward_pass_captured_beside_an_eager_graph_is_an_error():
    x, kernel = make((20, 64), "f32", 1).cuda().requires_grad_(), make((64, 30), "f32", 2).cuda().requires_grad_()
    alive = math_ops.lineari8(x, kernel)  # noqa: F841
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="made on the default stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            math_ops.lineari8(x, kernel).backward(torch.ones(20, 30, device="cuda"))
    torch.cuda.synchronize()


def test_calls_without_a_gradient_refuse_what_requires_one():
    x, kernel = make((5, 40), "f32", 1).cuda().requires_grad_(), make((40, 30), "f32", 2).cuda()
    w, bias = functors.int8_quantize(kernel, 0), torch.ones(30, device="cuda", requires_grad=True)
    for call in (lambda: functors.int8_linear(x, w), lambda: functors.int8_linear(x.detach(), w, bias), lambda: functors.int8_matmul(w, w, bias)):
        with pytest.raises(RuntimeError, match="requires one"):
            call()
        with torch.no_grad():
            call()
    g, = torch.autograd.grad(math_ops.lineari8(x, kernel).sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError, match="are not provided"):
        g.sum().backward()


@pytest.mark.parametrize("call,error", [
    (lambda x, w: functors.int8_quantize(x, 2), ValueError), (lambda x, w: functors.int8_quantize(x.double()), TypeError), (lambda x, w: functors.int8_quantize(x[0]), ValueError),
    (lambda x, w: functors.int8_quantize(x[:0]), ValueError), (lambda x, w: functors.int8_linear(x[:, 1:], w), ValueError), (lambda x, w: functors.int8_linear(x, x), TypeError),
    (lambda x, w: functors.int8_linear(x, w, torch.ones(29, device="cuda")), ValueError), (lambda x, w: functors.int8_linear(x, w, activation="gelu"), ValueError),
    (lambda x, w: functors.int8_linear(x, functors.I8Tensor(w.data, 31, 40)), ValueError), (lambda x, w: functors.int8_linear(x, functors.I8Tensor(w.data[1:], 30, 40)), ValueError),
    (lambda x, w: functors.int8_matmul(w, functors.int8_quantize(x[:, 1:].contiguous())), ValueError), (lambda x, w: functors.int8_matmul(w, w, dtype=torch.int8), TypeError),
    (lambda x, w: functors.int8_dequantize(w, torch.float64), TypeError), (lambda x, w: math_ops.lineari8(x, torch.ones(39, 5, device="cuda")), ValueError),
    (lambda x, w: math_ops.lineari8(x, torch.ones(40, 0, device="cuda")), ValueError), (lambda x, w: math_ops.lineari8(x, torch.ones(40, 5)), TypeError),
    (lambda x, w: math_ops.lineari8(x, torch.ones(40, 5, device="cuda"), torch.ones(4, device="cuda")), ValueError),
    (lambda x, w: functors.int8_quantize(torch.ones(1, device="cuda").expand(1, (1 << 21) + 1)), ValueError)])
def test_refusals(call, error):
    x = make((5, 40), "f32", 1).cuda()
    with pytest.raises(error):
        call(x, functors.int8_quantize(make((40, 30), "f32", 2).cuda(), 0))


# ---- layers, together as they are used -----------------------------------------------------------------------------

def test_layer_and_its_packed_form():
    for activation in (None, "relu", "gelu", "swish", "tanh"):
        layer = layers.densei8(70, activation, input_dim=200).cuda()
        with torch.no_grad():
            layer.bias.normal_()
        x = make((6, 5, 200), "bf16", 1).cuda().requires_grad_()
        y = layer(x)
        y.float().square().sum().backward()
        assert y.shape == (6, 5, 70) and x.grad.dtype == torch.bfloat16 and layer.kernel.grad.dtype == torch.float32
        served = layer.pack()
        with torch.no_grad():
            assert torch.equal(served(x), y)
            again = layers.packed_densei8(torch.zeros_like(layer.kernel), torch.zeros_like(layer.bias), layer.activation)
            again.load_state_dict(served.state_dict())
            assert torch.equal(again(x), y)
        with pytest.raises(RuntimeError, match="of width"):
            layers.packed_densei8(torch.zeros(201, 70, device="cuda"), torch.zeros(70, device="cuda")).load_state_dict(served.state_dict())


def test_what_a_layer_keeps_is_a_byte_for_each_value():
    layer = layers.densei8(256, "gelu", input_dim=512).cuda()
    x = make((1024, 512), "f32", 1).cuda().requires_grad_()
    sizes = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: sizes.append(t.numel() * t.element_size()) or t, lambda t: t):
        layer(x)
    kernel = 512 * 256 + 4 * 256
    assert sum(sizes) == 1024 * 512 + 4 * 1024 + kernel + 1024 * (256 + 4)


def test_an_encoder_s_dense_half_trains_and_serves():
    """Normalisation, two dense layers with an activation between, and the residual: gradients against the same block
    composed of the definitions in 64 bits, token by token of 8-bit operands."""
    torch.manual_seed(0)
    norm = layers.LayerNormalization(keep_bits=8, input_dim=96).cuda()
    up, down = layers.densei8(384, "gelu", input_dim=96).cuda(), layers.densei8(96, input_dim=384).cuda()
    x = torch.randn(4, 33, 96, device="cuda")

    def block(t):
        return t + down(up(norm(t)))

    leaf = x.clone().requires_grad_()
    y = block(leaf)
    dy = torch.randn_like(y) * 0.1
    params = [leaf, *norm.parameters(), *up.parameters(), *down.parameters()]
    grads = torch.autograd.grad(y, params, dy)
    exact = [p.detach().double().requires_grad_() for p in params]
    t, gamma, beta, wu, bu, wd, bd = exact
    n = torch.nn.functional.layer_norm(t, (96,), gamma, beta, 1e-3)
    want = t + torch.nn.functional.gelu(n @ wu + bu) @ wd + bd
    # 8 bits are off by half a step of 1 / 127 of a row's largest, 1 / 880 root mean square of it: some 0.4 percent of a normal row's
    # norm for each operand, eight operands deep at most
    for got, exactly in zip((y, *grads), (want, *torch.autograd.grad(want, exact, dy.double()))):
        assert ((got.double() - exactly).norm() / exactly.norm()) < 0.05
    served_up, served_down = up.pack(), down.pack()
    with torch.no_grad():
        assert torch.equal(x + served_down(served_up(norm(x))), block(x))
        token = x[:1, :1]
        assert torch.equal(token + served_down(served_up(norm(token))), block(x)[:1, :1])
    from approxtrain_amd.optimizers import AdamW
    opt = AdamW(params[1:], lr=1e-3)
    for _ in range(2):
        opt.zero_grad()
        block(x).square().mean().backward()
        opt.step()
    assert all(torch.isfinite(p).all() for p in params)


def test_products_on_another_stream():
    w = functors.int8_quantize(make((1000, 500), "f16", 1).cuda(), 0)
    xs = [make((m, 1000), "f16", m).cuda() for m in (1, 40, 700)]
    want = [functors.int8_linear(x, w) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(functors.int8_linear(x, w))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 3]) for i, g in enumerate(got))


def test_offsets_past_32_bits():
    """Operands of more than 2^32 bytes, results of more than 2^31 elements: their last rows are those of the rows by themselves."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(70016, 65536, dtype=torch.float16, device="cuda")  # 9.2 GB, 4.6 GB of codes
    x.normal_(generator=g)
    few = x[-64:].clone()
    w = functors.int8_quantize(torch.randn((65536, 20), device="cuda", generator=g), 0)
    q = functors.int8_quantize(x)
    assert q.nbytes() > 1 << 32
    want = functors.int8_linear(few, w)
    assert torch.equal(functors.int8_matmul(q, w, dtype=torch.float16)[-64:], want)
    assert torch.equal(functors.int8_linear(x, w)[-64:], want)
    assert torch.equal(q.dequantize(torch.float16)[-64:], functors.int8_quantize(few).dequantize(torch.float16))
    del q
    torch.cuda.empty_cache()
    by_columns = functors.int8_quantize(x, 0)  # the last columns', of all rows
    assert torch.equal(by_columns.dequantize(torch.float16)[-64:], functors.int8_quantize(x[:, -64:], 0).dequantize(torch.float16))
    del by_columns, x
    torch.cuda.empty_cache()
    a, b = torch.randn((70016, 64), device="cuda", generator=g), torch.randn((64, 40000), device="cuda", generator=g)
    wide = functors.int8_quantize(b, 0)
    assert torch.equal(functors.int8_linear(a.bfloat16(), wide)[-64:], functors.int8_linear(a[-64:].bfloat16(), wide))


def test_status_of_the_library_is_raised():
    with pytest.raises(AmsimError):
        from approxtrain_amd._lib import check
        check(load_library().amsim_i8_matmul(None, None, 4, 4, 4, None, 0, 0, 1 << 20, 0, None, 0, None))
