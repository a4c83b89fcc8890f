"""The 4-bit dense layer, its packed form, the optimizer class and the example that runs them together."""
import copy
import importlib.util
import os

import numpy as np
import pytest
import torch

from approxtrain_amd import functors, math_ops
from approxtrain_amd.layers import densemx, packed_densemx
from approxtrain_amd.optimizers import AdamW
from tests import mx_reference as ref

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def host64(t):
    return t.detach().double().cpu().numpy()


@pytest.mark.parametrize("activation", [None, "relu", "tanh"])
@pytest.mark.parametrize("shape", [(5, 40), (2, 3, 40), (40,)])
def test_layer_against_the_formula(shape, activation):
    torch.manual_seed(1)
    layer = densemx(24, activation, bias_initializer="ones").cuda()
    x = torch.randn(shape, device="cuda")
    y = layer(x)
    assert y.shape == shape[:-1] + (24,) and layer.kernel.shape == (40, 24)
    a, b = ref.mx_values(host64(x).reshape(-1, 40)), ref.mx_values(host64(layer.kernel), 0)
    z, mag = a @ b + 1.0, np.abs(a) @ np.abs(b) + 1.0
    want = {None: z, "relu": np.maximum(z, 0), "tanh": np.tanh(z)}[activation]
    # two blocks of 32 and the bias: three sums of 2^-23 each; tanh: 4 units in the last place
    assert (np.abs(host64(y).reshape(-1, 24) - want) <= 3 * 2.0 ** -23 * mag + 2.0 ** -21 * np.abs(want)).all()


def test_packed_layer_is_the_layer():
    torch.manual_seed(2)
    layer = densemx(33, "relu", input_dim=70).cuda()
    packed = layer.pack()
    assert isinstance(packed, packed_densemx) and not list(packed.parameters())
    for rows in (1, 20, 300):
        x = torch.randn(rows, 70, device="cuda")
        a, b = ref.mx_values(host64(x)), ref.mx_values(host64(layer.kernel), 0)
        tol = 2 * 4 * 2.0 ** -23 * (np.abs(a) @ np.abs(b) + np.abs(host64(layer.bias)))  # either side: three blocks and the bias
        assert (np.abs(host64(layer(x)) - host64(packed(x))) <= tol).all()
    assert torch.equal(packed(x.reshape(3, 100, 70)), packed(x).reshape(3, 100, 33))
    again = packed_densemx(torch.zeros_like(layer.kernel), torch.zeros_like(layer.bias), "relu")
    again.load_state_dict(packed.state_dict())
    assert torch.equal(again(x), packed(x))


def test_layer_refusals():
    with pytest.raises(ValueError, match="units"):
        densemx(0)
    with pytest.raises(ValueError, match="no weights"):
        densemx(4).pack()
    with pytest.raises(ValueError, match="activation"):
        densemx(4, "nothing")
    layer = densemx(4, input_dim=8).cuda()
    with pytest.raises(ValueError, match="linearmx"):
        layer(torch.zeros(2, 9, device="cuda"))
    with pytest.raises(TypeError, match="device memory"):
        layer.cpu()(torch.zeros(2, 8))


def test_dense_calls_refuse():
    x, w = torch.randn(70, 40, device="cuda"), torch.randn(40, 24, device="cuda")
    out, kept = functors.mxfp4_dense(x, w, activation="relu")
    g = torch.randn(70, 24, device="cuda")
    good = functors.mxfp4_dense_grad(g, kept, 70, 40, 24, out, torch.float32, torch.float32)
    assert [t.shape for t in good] == [(70, 40), (40, 24), (24,)]
    for bad in (dict(grad=g[:69]), dict(kept=kept[:-1]), dict(kept=kept.float()), dict(out=out[:, :23]), dict(out=out.bfloat16()), dict(units=25),
                dict(kernel_dtype=None), dict(need_x=False)):
        args = dict(grad=g, kept=kept, rows=70, width=40, units=24, out=out, kernel_dtype=torch.float32)
        args.update(bad)
        with pytest.raises(ValueError):
            functors.mxfp4_dense_grad(**args)
    with pytest.raises(TypeError, match="result"):
        functors.mxfp4_dense_grad(g, kept, 70, 40, 24, out, torch.float64)
    with pytest.raises(TypeError, match="device memory"):
        functors.mxfp4_dense_grad(g, kept.cpu(), 70, 40, 24, out, torch.float32)
    with pytest.raises(ValueError, match="rows"):
        functors.mxfp4_dense(x, w.t())
    with pytest.raises(TypeError, match="kernel"):
        functors.mxfp4_dense(x, w.long())


def test_an_operand_with_other_data_is_refused():
    q = functors.mxfp4_quantize(torch.randn(20, 300, device="cuda"))
    for bad in (functors.MXTensor(q.data[:-1], 20, 300), functors.MXTensor(q.data, 40, 300), functors.MXTensor(q.data.float(), 20, 300)):
        with pytest.raises(ValueError, match="data"):
            functors.mxfp4_dequantize(bad)
        with pytest.raises(ValueError, match="data"):
            functors.mxfp4_matmul(bad, functors.MXTensor(q.data, bad.rows, bad.length) if bad.rows == 20 else bad)


def test_gradients_of_gradients_say_that_they_are_missing():
    x, w = torch.randn(9, 40, device="cuda", requires_grad=True), torch.randn(40, 24, device="cuda", requires_grad=True)
    dy = torch.randn(9, 24, device="cuda", requires_grad=True)
    gx, gw = torch.autograd.grad(math_ops.linearmx(x, w), [x, w], dy, create_graph=True)
    with pytest.raises(RuntimeError, match="not provided"):
        (gx.sum() + gw.sum()).backward()
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises((TypeError, RuntimeError), match="forward|jvp"):
            math_ops.linearmx(torch.autograd.forward_ad.make_dual(x.detach(), x.detach()), w.detach())


@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (0, 1), (0, 2), (1, 2)])
def test_gradients_one_by_one_are_those_of_all(wanted):
    """(Each alone is planned by itself; these reductions are too short to be split.)"""
    leaves = [torch.randn(s, device="cuda").requires_grad_() for s in ((200, 96), (96, 130), (130,))]
    dy = torch.randn(200, 130, device="cuda")

    def grads(which):
        return torch.autograd.grad(math_ops.linearmx(*leaves, activation="relu"), [leaves[i] for i in which], dy)

    every = grads((0, 1, 2))
    for i, g in zip(wanted, grads(wanted)):
        assert torch.equal(g, every[i])


@pytest.mark.parametrize("m,width,units", [(8192, 96, 70), (100, 5000, 65), (66, 70, 9000), (20000, 40, 33)])
def test_split_reductions_of_a_backward_pass(m, width, units):
    """Long reductions beside short ones in the launch that they share, each against the product of its own operands."""
    x, w, dy = (torch.randn(s, device="cuda") for s in ((m, width), (width, units), (m, units)))
    b = torch.zeros(units, device="cuda", requires_grad=True)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    gx, gw, gb = torch.autograd.grad(math_ops.linearmx(xl, wl, b), [xl, wl, b], dy)
    (xr, xc), (wr, wc), (gr, gc) = (functors.mxfp4_quantize_both(t) for t in (x, w, dy))
    for got, p, q in ((gx, gr, wr), (gw, xc, gc)):
        a, c = p.dequantize().double(), q.dequantize().double()
        tol = (-(-p.length // 32) + 18) * 2.0 ** -23 * (a.abs() @ c.abs().t())
        assert bool(((got.double() - a @ c.t()).abs() <= tol).all())
    # runs of up to 32 in 32 bits, those added in 16 runs of ceil(m / 512), those in order
    assert bool(((gb.double() - dy.double().sum(0)).abs() <= (32 + -(-m // 512) + 16) * 2.0 ** -24 * dy.double().abs().sum(0)).all())


@pytest.mark.parametrize("m", [1, 15, 16, 17, 32, 33, 64, 65])
@pytest.mark.parametrize("k", [32, 2048, 2049, 2600, 32768, 32800])
def test_few_rows_at_the_borders_of_their_kernels(m, k):
    x, w = torch.randn(m, k, device="cuda"), torch.randn(k, 35, device="cuda")
    q = functors.mxfp4_quantize(w, axis=0)
    got = functors.mxfp4_linear(x, q)
    a, c = functors.mxfp4_quantize(x).dequantize().double(), q.dequantize().double()
    tol = (-(-k // 32) + 18) * 2.0 ** -23 * (a.abs() @ c.abs().t())
    assert bool(((got.double() - a @ c.t()).abs() <= tol).all())
    assert bool(((functors.mxfp4_matmul(functors.mxfp4_quantize(x), q).double() - a @ c.t()).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(17, 10, 1), (31, 33, 33), (33, 100, 130), (50, 64, 500), (64, 1000, 128), (64, 17, 512), (18, 35, 1700)])
def test_some_tens_of_rows_converted_on_the_way(m, n, k, dtype):
    x, w, bias = torch.randn(m, k, device="cuda").to(dtype), torch.randn(k, n, device="cuda"), torch.randn(n, device="cuda")
    q = functors.mxfp4_quantize(w, axis=0)
    got = functors.mxfp4_linear(x, q, bias, "relu")
    assert got.dtype == dtype
    a, c, b = functors.mxfp4_quantize(x).dequantize().double(), q.dequantize().double(), bias.double()
    want, size = torch.relu(a @ c.t() + b), a.abs() @ c.abs().t() + b.abs()
    # sums in 32 bits, a rounding to the result's type, and of float16's small results half its smallest step
    tol = (-(-k // 32) + 19) * 2.0 ** -23 * size + want * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert bool(((got.double() - want).abs() <= tol).all())
    wide = torch.full((m, k + 3), float("nan"), device="cuda", dtype=dtype)
    wide[:, 1:k + 1] = x
    assert torch.equal(functors.mxfp4_linear(wide[:, 1:k + 1], q, bias, "relu"), got)
    wide[m - 1, k] = float("inf")
    bad = torch.isnan(functors.mxfp4_linear(wide[:, 1:k + 1], q))
    assert bool(bad[m - 1].all()) and not bool(bad[:m - 1].any())


@pytest.mark.parametrize("m,n,k", [(256, 33000, 130), (2100, 2300, 1100), (1500, 2500, 300), (4097, 4095, 700), (300, 40000, 64)])
def test_products_in_each_tile(m, n, k):
    """Odd extents in tiles of 256 x 256, 256 x 128 and 128, with a bias and results of 16 bits."""
    x, w, bias = torch.randn(m, k, device="cuda"), torch.randn(n, k, device="cuda"), torch.randn(n, device="cuda")
    p, q = functors.mxfp4_quantize(x), functors.mxfp4_quantize(w)
    a, c = p.dequantize().double(), q.dequantize().double()
    z = a @ c.t() + bias.double()
    tol = (-(-k // 32) + 3) * 2.0 ** -23 * (a.abs() @ c.abs().t() + bias.double().abs())
    assert bool(((functors.mxfp4_matmul(p, q, bias).double() - z).abs() <= tol).all())
    got = functors.mxfp4_matmul(p, q, bias, "relu", torch.bfloat16).double()
    z = z.clamp(min=0)
    assert bool(((got - z).abs() <= tol * 1.01 + 2.0 ** -8 * z.abs()).all())


@pytest.mark.parametrize("dtype,m,n", [(torch.float32, 7300, 8201), (torch.bfloat16, 14500, 8203), (torch.float16, 440, 270001)])
def test_results_larger_than_the_cache(dtype, m, n):
    """More than 224 MB of results, the last rows' and columns' tiles not full."""
    k = 200
    x, w, bias = torch.randn(m, k, device="cuda"), torch.randn(k, n, device="cuda"), torch.randn(n, device="cuda")
    a, c = functors.mxfp4_quantize(x), functors.mxfp4_quantize(w, axis=0)
    got = functors.mxfp4_matmul(a, c, bias, "relu", dtype=dtype)
    left, right = a.dequantize(torch.float32).double(), c.dequantize(torch.float32).double().t()
    for rows in torch.arange(m, device="cuda").split(500):
        want, size = torch.relu(left[rows] @ right + bias.double()), left[rows].abs() @ right.abs() + bias.double().abs()
        tol = (-(-k // 32) + 19) * 2.0 ** -23 * size + want * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert bool(((got[rows].double() - want).abs() <= tol).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_steps_as_the_function_does_and_goes_on_from_a_saved_state(bits):
    torch.manual_seed(3)
    params = [torch.nn.Parameter(torch.randn(s, device="cuda", dtype=t)) for s, t in (((30, 40), torch.float32), ((7,), torch.bfloat16), ((300,), torch.float32))]
    alone = [p.detach().clone() for p in params]
    states = [functors.AdamWState([alone[0], alone[2]], bits), functors.AdamWState([alone[1]], bits)]
    opt = AdamW(params, lr=1e-2, weight_decay=0.1, state_bits=bits)
    scale = torch.tensor([0.5], device="cuda")
    for step in (1, 2, 3):
        grads = [torch.randn_like(p) for p in params]
        for p, g in zip(params, grads):
            p.grad = g
        if step == 3:
            params[0].grad = grads[0].t().contiguous().t()   # (not contiguous)
            saved = copy.deepcopy(opt.state_dict())
            other = [torch.nn.Parameter(p.detach().clone()) for p in params]
            for p, g in zip(other, grads):
                p.grad = g
            resumed = AdamW(other, lr=1.0, state_bits=bits)
            resumed.load_state_dict(saved)
            resumed.step(grad_scale=scale)
        opt.step(grad_scale=scale)
        functors.adamw_step(states[0], [grads[0], grads[2]], step, 1e-2, 0.9, 0.999, 1e-8, 0.1, scale)
        functors.adamw_step(states[1], [grads[1]], step, 1e-2, 0.9, 0.999, 1e-8, 0.1, scale)
        for p, a in zip(params, alone):
            assert torch.equal(p, a)
    for p, o in zip(params, other):
        assert torch.equal(p, o)
    with pytest.raises(ValueError, match="bits"):
        AdamW(params, state_bits=40 - bits).load_state_dict(saved)
    with pytest.raises(ValueError, match="other parameters"):
        AdamW(params[:2], state_bits=bits).load_state_dict(saved)
    with pytest.raises(ValueError, match="state_bits"):
        AdamW(params, state_bits=4)


def test_capture_beside_a_living_graph_of_the_same_leaves():
    """A graph made on the default stream holds the nodes that add its leaves' gradients there: a captured backward pass is
    refused while it lives, and works and replays once it is gone."""
    x, w = torch.randn(40, 70, device="cuda"), torch.randn(70, 30, device="cuda", requires_grad=True)
    b = torch.zeros(30, device="cuda", requires_grad=True)
    leaves = [w, b]

    def step():
        return torch.autograd.grad(math_ops.linearmx(x, w, b, activation="relu").sum(), leaves)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    living = math_ops.linearmx(x, w, b)
    with pytest.raises(RuntimeError, match="lives"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    torch.cuda.synchronize()
    for got, want in zip(torch.autograd.grad(living.sum(), leaves, retain_graph=True), torch.autograd.grad(math_ops.linearmx(x, w, b).sum(), leaves)):
        assert torch.equal(got, want)
    del living
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        with torch.no_grad():
            w.normal_(generator=torch.Generator(device="cuda").manual_seed(seed))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(captured, step()):
            assert torch.equal(got, want)


def test_optimizer_in_a_graph():
    """A captured step, replayed with eager work between, steps as eager calls of the same number do."""
    p = [torch.randn(n, device="cuda") for n in (5, 300, 4097)]
    g = [torch.randn_like(t) for t in p]
    q, state, eager = [t.clone() for t in p], functors.AdamWState(p, 8), None
    eager = functors.AdamWState(q, 8)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        functors.adamw_step(state, g, 7)
    for _ in range(3):
        for t in g:
            t.normal_()
        graph.replay()
        torch.cuda.synchronize()
        functors.adamw_step(eager, g, 7)
        for a, b in zip(p + [state.m, state.v, state.m_scale, state.v_scale], q + [eager.m, eager.v, eager.m_scale, eager.v_scale]):
            assert torch.equal(a, b)


def test_moments_of_other_buffers_are_refused():
    p, g = torch.zeros(600, device="cuda"), torch.ones(600, device="cuda")
    for name in ("m", "v_scale"):
        state = functors.AdamWState([p], 8)
        setattr(state, name, getattr(state, name)[:-1])
        with pytest.raises(ValueError, match="buffers"):
            functors.adamw_step(state, [g], 1)
        with pytest.raises(ValueError, match="blocks of 256"):
            state.first_moments() if name == "m" else state.second_roots()
    assert not p.any()


@pytest.mark.parametrize("bits", [8, 32])
def test_example_learns(bits):
    spec = importlib.util.spec_from_file_location("lenet300_mx", os.path.join(ROOT, "examples", "lenet300_mx.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    _, _, losses, (trained, served) = example.train(steps=120, state_bits=bits)
    assert losses[-1] < 0.5 * losses[0] and trained > 0.9 and abs(trained - served) < 0.02
