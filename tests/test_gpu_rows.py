"""Layer normalisation, activations that keep their input in 8 bits, and the keeping, against their definitions in 64 bits;
``rows_reference`` derives the tolerances."""
import pytest
import torch

from approxtrain_amd import functors, layers, math_ops
from tests import rows_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# every way that a row lies over lanes, with its borders, and rows that no workgroup holds
COLS = [1, 2, 7, 15, 16, 17, 64, 127, 128, 129, 300, 511, 512, 513, 1000, 1024, 1025, 2047, 2048, 2049, 4095, 4096, 4097, 8192, 8193, 16383, 16384,
        16385, 40001]


def make(rows, cols, dtype, seed, offset=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, cols), generator=g) * torch.exp(0.5 * torch.randn(cols, generator=g)) + offset
    return x.to(DTYPES[dtype])


def vectors(cols, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (1 + 0.3 * torch.randn(cols, generator=g)).to(dtype), (0.3 * torch.randn(cols, generator=g)).to(dtype)


def close(got, want, tol, name):
    half, tiny = ref.half_step(got.dtype), torch.finfo(got.dtype).smallest_normal * ref.half_step(got.dtype) * 2
    got, want = got.detach().double().cpu(), want.cpu()
    assert got.shape == want.shape, name
    tol = tol.cpu() + half * want.abs() * 1.01 + tiny
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} outside; worst {float(((got - want).abs() / tol).max()):.3g} of the tolerance"


def kept_of(x):
    return ref.int8_values(x).float()  # (a code times its scale, rounded once)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", COLS)
def test_kept_values_are_the_definition_s(cols, dtype):
    x = make(9, cols, dtype, cols)
    x[1] = 0
    x[2] *= 1e-4
    x[3, 0] = x[3].abs().max() * 1.5
    k = functors.keep8(x.cuda())
    assert k.nbytes() == 9 * (-(-cols // 16) * 16 + 4)
    assert torch.equal(k.values(torch.float32).cpu(), kept_of(x))
    assert torch.equal(k.values().cpu(), kept_of(x).to(x.dtype)) and k.values().dtype == x.dtype


def test_codes_at_ties_and_at_the_ends_of_the_range():
    # multipliers that are exact: 127 / 127 and its powers of two, so that halves tie to the even integer
    row = torch.cat([torch.tensor([127.0]), torch.arange(-126.5, 127.0, 1.0)])
    x = torch.stack([row * 2.0 ** e for e in (-100, -20, 0, 50, 120)])
    assert torch.equal(functors.keep8(x.cuda()).values().cpu(), torch.round(row) * 2.0 ** torch.tensor([-100.0, -20, 0, 50, 120])[:, None])
    # below 2^-119 the step is that of 2^-119; zeros stay zeros
    x = torch.tensor([[2.0 ** -130, 0.0], [2.0 ** -149, 2.0 ** -140], [0.0, -0.0], [2.0 ** -119, 2.0 ** -120], [3.0e38, -1.0e38]])
    assert torch.equal(functors.keep8(x.cuda()).values().cpu(), kept_of(x))


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("cols", [5, 700, 5000, 20000])
def test_a_row_that_is_not_finite_reads_back_as_nan(cols, bad):
    x = make(4, cols, "f32", 1)
    x[2, cols // 2] = bad
    got = functors.keep8(x.cuda()).values().cpu()
    assert torch.isnan(got[2]).all()
    keep = [0, 1, 3]
    assert torch.equal(got[keep], kept_of(x)[keep])


def check_norm(x, gamma, beta, dy, keep_bits, epsilon=1e-3):
    """All of a training step against the definition; returns what came out."""
    leaves = [t.cuda().requires_grad_() if t is not None else None for t in (x, gamma, beta)]
    y = math_ops.layernorm(*leaves, epsilon=epsilon, keep_bits=keep_bits)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy.cuda())
    kept = kept_of(x) if keep_bits == 8 else None
    want = ref.layer_norm(x, gamma, beta, epsilon, dy, kept)
    tol = ref.layer_norm_tolerances(x, gamma, beta, epsilon, dy, kept)
    close(y, want[0], tol[0], "y")
    names = iter(grads)
    for i, (t, name) in enumerate(((x, "dx"), (gamma, "dgamma"), (beta, "dbeta"))):
        if t is not None:
            g = next(names)
            assert g.dtype == t.dtype
            close(g, want[i + 1], tol[i + 1], name)
    with torch.no_grad():
        assert torch.equal(functors.layer_norm(*leaves, epsilon=epsilon), y)
    return (y, *grads)


@pytest.mark.parametrize("keep_bits", [None, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", COLS)
def test_layer_norm_over_widths(cols, dtype, keep_bits):
    rows = 21 if cols <= 4096 else 5
    x = make(rows, cols, dtype, cols)
    check_norm(x, *vectors(cols, 3), make(rows, cols, dtype, cols + 1), keep_bits)


@pytest.mark.parametrize("keep_bits", [None, 8])
@pytest.mark.parametrize("rows,cols", [(1, 512), (2, 300), (3, 4096), (65, 128), (4099, 96), (9001, 8), (2600, 520), (1300, 3000), (700, 8200), (130, 17000)])
def test_layer_norm_over_rows(rows, cols, keep_bits):
    check_norm(make(rows, cols, "bf16", 1), *vectors(cols, 3), make(rows, cols, "bf16", 2), keep_bits)


@pytest.mark.parametrize("params", ["none", "gamma", "beta"])
def test_layer_norm_without_parameters(params):
    gamma, beta = vectors(700, 3)
    check_norm(make(33, 700, "f32", 1), gamma if params == "gamma" else None, beta if params == "beta" else None, make(33, 700, "f32", 2), None)


@pytest.mark.parametrize("param", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_of_every_pair_of_types(dtype, param):
    check_norm(make(40, 1003, dtype, 1), *vectors(1003, 3, DTYPES[param]), make(40, 1003, dtype, 2), None)


@pytest.mark.parametrize("offset", [30.0, -500.0])
def test_layer_norm_far_from_zero(offset):
    check_norm(make(17, 2000, "f32", 1, offset), *vectors(2000, 3), make(17, 2000, "f32", 2), None)


def test_layer_norm_of_constant_rows_and_epsilon_zero():
    x = torch.full((5, 40), 3.0)
    gamma, beta = vectors(40, 3)
    y = functors.layer_norm(x.cuda(), gamma.cuda(), beta.cuda())
    assert torch.equal(y.cpu(), beta.expand(5, 40))
    check_norm(make(5, 40, "f32", 1), gamma, beta, make(5, 40, "f32", 2), None, epsilon=0.0)


def test_layer_norm_of_strided_and_higher_rank_tensors():
    base = make(48, 700, "f16", 1).cuda()
    gamma, beta = (t.cuda() for t in vectors(600, 3))
    for view in (base[:, 100:], base[::3, 50:650], make(600, 48, "f16", 2).cuda().t(), base[:, 100:].reshape(4, 12, 600), base[:1, 3:603].expand(7, 600)):
        x = view.detach().requires_grad_()
        plain = view.detach().clone(memory_format=torch.contiguous_format).requires_grad_()
        dy = make(view.numel() // 600, 600, "f16", 5).cuda().reshape(view.shape)
        for keep in (None, 8):
            a = math_ops.layernorm(x, gamma, beta, keep_bits=keep)
            b = math_ops.layernorm(plain, gamma, beta, keep_bits=keep)
            assert a.shape == view.shape and a.is_contiguous() and torch.equal(a, b)
            ga, = torch.autograd.grad(a, [x], torch.stack([dy, dy], -1)[..., 0])
            gb, = torch.autograd.grad(b, [plain], dy)
            assert torch.equal(ga, gb)
    one = torch.randn(600).cuda()
    assert torch.equal(functors.layer_norm(one, gamma, beta), functors.layer_norm(one[None], gamma, beta)[0])


def test_layer_norm_of_no_rows():
    x = torch.empty(0, 8, device="cuda", requires_grad=True)
    gamma = torch.ones(8, device="cuda", requires_grad=True)
    y = math_ops.layernorm(x, gamma, torch.zeros(8, device="cuda"))
    gx, gg = torch.autograd.grad(y, [x, gamma], torch.empty(0, 8, device="cuda"))
    assert y.shape == gx.shape == (0, 8) and torch.equal(gg, torch.zeros_like(gamma))
    z = torch.empty(2, 0, 8, device="cuda", requires_grad=True)
    assert math_ops.layernorm(z, gamma).shape == (2, 0, 8) and functors.layer_norm(z.detach()).shape == (2, 0, 8)


def test_layer_norm_keeps_nan_in_its_row():
    x = make(6, 800, "f32", 1)
    x[3, 7] = float("nan")
    x[4, 9] = float("inf")
    gamma, beta = vectors(800, 3)
    dy = make(6, 800, "f32", 2).cuda()
    for keep in (None, 8):
        leaf = x.cuda().requires_grad_()
        y = math_ops.layernorm(leaf, gamma.cuda(), beta.cuda(), keep_bits=keep)
        g, = torch.autograd.grad(y, [leaf], dy)
        for t in (y, g):
            assert torch.isnan(t[3]).all() and not torch.isfinite(t[4]).any() and torch.isfinite(t[[0, 1, 2, 5]]).all()


def test_layer_norm_asked_for_some_gradients():
    x, dy = make(70, 900, "bf16", 1).cuda(), make(70, 900, "bf16", 2).cuda()
    gamma, beta = (t.cuda() for t in vectors(900, 3))
    everything = [t.clone().requires_grad_() for t in (x, gamma, beta)]
    want = torch.autograd.grad(math_ops.layernorm(*everything), everything, dy)
    for which in range(1, 8):
        leaves = [t.clone().requires_grad_(bool(which >> i & 1)) for i, t in enumerate((x, gamma, beta))]
        asked = [t for t in leaves if t.requires_grad]
        got = iter(torch.autograd.grad(math_ops.layernorm(*leaves), asked, dy))
        for i in range(3):
            if which >> i & 1:
                assert torch.equal(next(got), want[i])
    for i in range(3):
        assert torch.equal(torch.autograd.grad(math_ops.layernorm(*everything), [everything[i]], dy)[0], want[i])


# ---- activations ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["gelu", "swish"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", COLS)
def test_activations(cols, dtype, kind):
    rows = 13 if cols <= 4096 else 3
    x, dy = make(rows, cols, dtype, cols), make(rows, cols, dtype, cols + 1)
    leaf = x.cuda().requires_grad_()
    y = math_ops.activationi8(leaf, kind)
    g, = torch.autograd.grad(y, [leaf], dy.cuda())
    value, slope = ref.ACTIVATIONS[kind]
    kept = kept_of(x)
    tol_y, tol_slope = ref.activation_tolerances(kind, x, kept)
    close(y, value(x.double()), tol_y, "y")
    want = dy.double() * slope(kept.double())
    close(g, want, dy.double().abs() * tol_slope + ref.U * want.abs(), "dx")
    with torch.no_grad():
        assert torch.equal(math_ops.activationi8(leaf, kind), y)


@pytest.mark.parametrize("kind", ["gelu", "swish"])
def test_activations_over_their_range(kind):
    x = torch.cat([torch.linspace(-30, 30, 60001), torch.tensor([-1e4, 1e4, -120.0, 120.0, 0.0, 1e-30, -1e-30])])[None]
    value, slope = ref.ACTIVATIONS[kind]
    small = x[:, :60001]
    tol, _ = ref.activation_tolerances(kind, x, x)
    close(math_ops.activationi8(x.cuda(), kind), value(x.double()), tol, "y")
    leaf = small.cuda().requires_grad_()
    g, = torch.autograd.grad(math_ops.activationi8(leaf, kind), [leaf], torch.ones_like(leaf))
    kept = kept_of(small)
    _, tol = ref.activation_tolerances(kind, small, kept)
    close(g, slope(kept.double()), tol, "slope")


@pytest.mark.parametrize("kind,plain", [("gelu", torch.nn.functional.gelu), ("swish", torch.nn.functional.silu)])
def test_activations_at_infinities(kind, plain):
    x = torch.tensor([[float("inf"), 1.0], [float("-inf"), 1.0], [float("nan"), 1.0]]).cuda().requires_grad_()
    y = math_ops.activationi8(x, kind)
    want = plain(x.detach())
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.isinf(y), torch.isinf(want))
    assert torch.isnan(torch.autograd.grad(y, [x], torch.ones_like(x))[0]).all()  # (rows that have no scale)


def test_activations_of_strided_and_empty_tensors():
    base = make(48, 700, "bf16", 1).cuda()
    for view in (base[:, 100:], base[::3, 50:650], base.t(), base[:, 100:].reshape(4, 12, 600)):
        a, b = view.detach().requires_grad_(), view.detach().clone(memory_format=torch.contiguous_format).requires_grad_()
        ya, yb = math_ops.activationi8(a, "gelu"), math_ops.activationi8(b, "gelu")
        dy = torch.randn(view.shape, device="cuda").to(view.dtype)
        assert ya.shape == view.shape and torch.equal(ya, yb)
        assert torch.equal(torch.autograd.grad(ya, [a], dy)[0], torch.autograd.grad(yb, [b], dy.transpose(0, 1).contiguous().transpose(0, 1))[0])
    z = torch.empty(0, 8, device="cuda", requires_grad=True)
    y = math_ops.activationi8(z, "swish")
    assert y.shape == (0, 8) and torch.autograd.grad(y, [z], torch.empty(0, 8, device="cuda"))[0].shape == (0, 8)


# ---- as a program uses them -----------------------------------------------------------------------------------------

def test_results_do_not_depend_on_what_runs_beside():
    x, dy = make(3000, 1027, "f16", 1).cuda(), make(3000, 1027, "f16", 2).cuda()
    gamma, beta = (t.cuda().requires_grad_() for t in vectors(1027, 3))
    leaf = x.clone().requires_grad_()

    def step(keep):
        y = math_ops.layernorm(leaf, gamma, beta, keep_bits=keep)
        z = math_ops.activationi8(y, "gelu")
        return (z, *torch.autograd.grad(z, [leaf, gamma, beta], dy))

    want = {k: step(k) for k in (None, 8)}
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 3]):
            got.append((8 if i % 2 else None, step(8 if i % 2 else None)))
    torch.cuda.synchronize()
    for k, outs in got:
        assert all(torch.equal(a, b) for a, b in zip(outs, want[k]))


def test_captured_training_steps():
    gamma, beta = (t.cuda().requires_grad_() for t in vectors(520, 3))
    xs = [make(100, 520, "f32", s).cuda() for s in range(4)]
    dy = make(100, 520, "f32", 9).cuda()
    leaf = xs[0].clone().requires_grad_()

    def step():
        y = math_ops.activationi8(math_ops.layernorm(leaf, gamma, beta, keep_bits=8), "swish")
        return (y.detach(), *torch.autograd.grad(y, [leaf, gamma, beta], dy))

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
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_backward_pass_captured_beside_an_eager_graph_is_an_error():
    x = make(20, 64, "f32", 1).cuda().requires_grad_()
    gamma = torch.ones(64, device="cuda", requires_grad=True)
    dy = torch.ones(20, 64, device="cuda")
    for call in (lambda: math_ops.layernorm(x, gamma), lambda: math_ops.activationi8(x, "gelu")):
        alive = call()  # noqa: F841
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="made on the default stream"):
            with torch.cuda.graph(graph):
                call().backward(dy)
        torch.cuda.synchronize()
        del alive


def test_a_captured_gradient_beside_an_eager_graph_of_leaves_that_are_not_asked_for():
    x = make(20, 64, "f32", 1).cuda()
    gamma = torch.ones(64, device="cuda", requires_grad=True)
    beta = torch.zeros(64, device="cuda", requires_grad=True)
    alive = (gamma * 1, beta * 1)  # noqa: F841  (their gradients would be added on the default stream)
    dy = torch.randn(20, 64, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        leaf = x.clone().requires_grad_()
        want = torch.autograd.grad(math_ops.layernorm(leaf, gamma, beta), [leaf], dy)[0]
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        got, = torch.autograd.grad(math_ops.layernorm(leaf, gamma, beta), [leaf], dy)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_gradients_of_gradients_are_refused():
    x = make(5, 40, "f32", 1).cuda().requires_grad_()
    for y in (math_ops.layernorm(x), math_ops.activationi8(x, "gelu")):
        g, = torch.autograd.grad(y.sum(), [x], create_graph=True)
        with pytest.raises(RuntimeError, match="are not provided"):
            g.sum().backward()


def test_calls_without_a_gradient_refuse_what_requires_one():
    x = make(5, 40, "f32", 1).cuda().requires_grad_()
    for call in (lambda: functors.layer_norm(x), lambda: functors.layer_norm(x.detach(), torch.ones(40, device="cuda", requires_grad=True)),
                 lambda: functors.keep8(x)):
        with pytest.raises(RuntimeError, match="requires one"):
            call()
        with torch.no_grad():
            call()


@pytest.mark.parametrize("call,error", [
    (lambda x: functors.layer_norm(x.double()), TypeError), (lambda x: functors.layer_norm(x[:, :0]), ValueError),
    (lambda x: functors.layer_norm(x, torch.ones(39, device="cuda")), ValueError), (lambda x: functors.layer_norm(x, torch.ones(40)), TypeError),
    (lambda x: functors.layer_norm(x, torch.ones(40, device="cuda"), torch.ones(40, device="cuda").half()), TypeError),
    (lambda x: functors.layer_norm(x, epsilon=-1.0), ValueError), (lambda x: functors.layer_norm(x, epsilon=float("nan")), ValueError),
    (lambda x: math_ops.layernorm(x, keep_bits=4), ValueError), (lambda x: math_ops.activationi8(x, "relu"), ValueError),
    (lambda x: math_ops.activationi8(x.int(), "gelu"), TypeError), (lambda x: functors.keep8(x[:0]), ValueError),
    (lambda x: functors.keep8(torch.tensor(1.0, device="cuda")), ValueError), (lambda x: functors.kept8_values(x), TypeError)])
def test_refusals(call, error):
    with pytest.raises(error):
        call(make(5, 40, "f32", 1).cuda())


def test_what_comes_back_in_another_form_is_refused():
    x = make(20, 64, "f32", 1).cuda().requires_grad_()
    for call in (lambda: math_ops.layernorm(x), lambda: math_ops.layernorm(x, keep_bits=8), lambda: math_ops.activationi8(x, "gelu")):
        for other in (lambda t: t[:-1], lambda t: t.cpu(), lambda t: t.double()):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, other):
                out = call()
            with pytest.raises((RuntimeError, TypeError)):
                out.sum().backward()


@pytest.mark.parametrize("cols", [8192, 20000])
def test_offsets_past_32_bits(cols):
    """Tensors of more than 2^32 elements: their last rows are those of the rows by themselves."""
    rows = (1 << 32) // cols + 100
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    few = x[-50:].clone()
    gamma, beta = (t.cuda() for t in vectors(cols, 3))
    assert torch.equal(functors.layer_norm(x, gamma, beta)[-50:], functors.layer_norm(few, gamma, beta))
    assert torch.equal(functors.keep8(x).values()[-50:], functors.keep8(few).values())
    for call in (lambda t: math_ops.layernorm(t, gamma, beta, keep_bits=8), lambda t: math_ops.layernorm(t, gamma, beta), lambda t: math_ops.activationi8(t, "swish")):
        a, b = x.requires_grad_(), few.requires_grad_()
        big, = torch.autograd.grad(call(a), [a], x.detach())
        assert torch.equal(big[-50:], torch.autograd.grad(call(b), [b], few.detach())[0])
        del big


def test_layer():
    layer = layers.LayerNormalization(keep_bits=8)
    x = make(30, 200, "bf16", 1).cuda().requires_grad_()
    y = layer(x)
    assert layer.gamma.shape == layer.beta.shape == (200,) and y.dtype == x.dtype and layer.gamma.device == x.device
    y.float().square().sum().backward()
    assert x.grad.dtype == torch.bfloat16 and layer.gamma.grad.dtype == layer.beta.grad.dtype == torch.float32
    bare = layers.LayerNormalization(center=False, scale=False, epsilon=1e-5)
    assert not list(bare.parameters())
    assert torch.equal(bare(x.detach()), functors.layer_norm(x.detach(), epsilon=1e-5))
