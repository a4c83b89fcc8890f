"""Layer normalisation and rows kept in 8 bits without a device: refusals of the C entries, which come back before any
kernel could run, and the tests' own definitions against differences."""
import pytest
import torch

from approxtrain_amd import functors, layers, load_library, math_ops
from tests import rows_reference as ref

A = 1 << 20  # an address that is never read


def lib():
    return load_library()


def test_sizes():
    size = lib().amsim_kept8_workspace_bytes
    assert size(1, 1) == 20 and size(3, 16) == 3 * 20 and size(3, 17) == 3 * 36 and size(0, 4) == size(4, 0) == size(-1, 4) == size(1 << 31, 1) == 0
    ws = lib().amsim_layer_norm_grad_workspace_bytes
    assert ws(1, 1) == 8 and ws(0, 4) == ws(4, -1) == 0 and ws(1 << 20, 4096) == 768 * 2 * 4096 * 4


def norm(x=A, dtype=0, rows=4, cols=4, stride=4, gamma=A, beta=A, param=0, eps=1e-3, out=A, stats=A, kept=A):
    return lib().amsim_layer_norm(x, dtype, rows, cols, stride, gamma, beta, param, eps, out, stats, kept, None)


@pytest.mark.parametrize("bad,status", [
    (dict(x=None), 1), (dict(out=None), 1), (dict(dtype=3), 1), (dict(dtype=-1), 1), (dict(param=7), 1), (dict(rows=0), 1), (dict(cols=0), 1), (dict(stride=3), 1),
    (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1), (dict(x=A + 2), 1), (dict(x=A + 1, dtype=1), 1), (dict(out=A + 2), 1), (dict(stats=A + 2), 1),
    (dict(kept=A + 8), 1), (dict(gamma=A + 2), 1), (dict(beta=A + 1, param=2), 1), (dict(rows=-1), 6), (dict(rows=1 << 31), 6), (dict(cols=1 << 31), 6),
    (dict(rows=1 << 30, cols=1 << 16, stride=1 << 16), 6)])
def test_layer_norm_refuses(bad, status):
    assert norm(**bad) == status


def norm_grad(grad=A, dtype=0, rows=4, cols=4, stride=4, x=A, x_stride=4, kept=None, stats=A, gamma=A, param=0, gx=A, gg=A, gb=A, ws=A, nbytes=1 << 20):
    return lib().amsim_layer_norm_grad(grad, dtype, rows, cols, stride, x, x_stride, kept, stats, gamma, param, gx, gg, gb, ws, nbytes, None)


@pytest.mark.parametrize("bad,status", [
    (dict(grad=None), 1), (dict(x=None), 1), (dict(kept=A), 1), (dict(stats=None), 1), (dict(dtype=3), 1), (dict(param=3), 1), (dict(stride=2), 1),
    (dict(x_stride=2), 1), (dict(x=None, kept=A + 4), 1), (dict(gx=A + 1), 1), (dict(gg=A + 2), 1), (dict(gb=A + 1, param=1), 1), (dict(ws=None), 5),
    (dict(ws=A + 128), 5), (dict(nbytes=31), 5), (dict(rows=0), 1), (dict(cols=1 << 31), 6), (dict(rows=1, cols=1 << 26, stride=1 << 26, x_stride=1 << 26), 6)])
def test_layer_norm_grad_refuses(bad, status):
    assert norm_grad(**bad) == status


def test_nothing_asked_for_is_nothing_done():
    assert norm_grad(gx=None, gg=None, gb=None, ws=None, nbytes=0) == 0


@pytest.mark.parametrize("args,status", [
    ((None, 0, 4, 4, 4, 2, A, A), 1), ((A, 0, 4, 4, 4, 1, A, A), 1), ((A, 0, 4, 4, 4, 9, A, A), 1), ((A, 0, 4, 4, 4, 2, None, None), 1), ((A, 0, 4, 4, 4, 2, A, A + 4), 1),
    ((A, 0, 4, 4, 4, 2, A + 2, A), 1), ((A, 5, 4, 4, 4, 2, A, A), 1), ((A, 0, 4, 4, 3, 2, A, A), 1), ((A, 0, 0, 4, 4, 2, A, A), 1), ((A, 0, 1 << 31, 4, 4, 2, A, A), 6)])
def test_activation_refuses(args, status):
    assert lib().amsim_activation(*args, None) == status


@pytest.mark.parametrize("args,status", [
    ((None, 0, 4, 4, 4, A, 2, A), 1), ((A, 0, 4, 4, 4, None, 2, A), 1), ((A, 0, 4, 4, 4, A, 2, None), 1), ((A, 0, 4, 4, 4, A, 0, A), 1), ((A, 0, 4, 4, 4, A, 1, A), 1),
    ((A, 0, 4, 4, 4, A + 4, 2, A), 1), ((A, 0, 4, 4, 4, A, 2, A + 1), 1), ((A, 3, 4, 4, 4, A, 2, A), 1)])
def test_activation_grad_refuses(args, status):
    assert lib().amsim_activation_grad(*args, None) == status


@pytest.mark.parametrize("args,status", [((None, 4, 4, 0, A), 1), ((A, 4, 4, 0, None), 1), ((A + 4, 4, 4, 0, A), 1), ((A, 4, 4, 3, A), 1), ((A, 0, 4, 0, A), 1)])
def test_kept8_values_refuses(args, status):
    assert lib().amsim_kept8_values(*args, None) == status


def test_host_tensors_are_refused():
    x = torch.ones(2, 4)
    for call in (lambda: functors.layer_norm(x), lambda: math_ops.layernorm(x), lambda: math_ops.activationi8(x, "gelu"), lambda: functors.keep8(x),
                 lambda: layers.LayerNormalization(input_dim=4)(x), lambda: functors.layer_norm(5), lambda: functors.keep8(None)):
        with pytest.raises(TypeError):
            call()


def test_layer_arguments():
    for bad in (dict(axis=0), dict(epsilon=-1), dict(keep_bits=16)):
        with pytest.raises(ValueError):
            layers.LayerNormalization(**bad)
    with pytest.raises(ValueError):
        math_ops.activationi8(torch.ones(1, 1), "tanh")


def test_the_definitions_gradients_against_differences():
    g = torch.Generator().manual_seed(0)
    x, dy, direction = (torch.randn((6, 11), generator=g, dtype=torch.float64) for _ in range(3))
    gamma, beta = torch.randn(11, generator=g, dtype=torch.float64), torch.randn(11, generator=g, dtype=torch.float64)
    _, dx, dgamma, dbeta = ref.layer_norm(x, gamma, beta, 1e-3, dy)
    h = 1e-6  # (central differences: off by h^2, and by 1e-16 / h)

    def along(f):
        return ((f(h) - f(-h)) * dy).sum() / (2 * h)

    v = torch.randn(11, generator=g, dtype=torch.float64)
    torch.testing.assert_close(along(lambda t: ref.layer_norm(x + t * direction, gamma, beta, 1e-3)), (dx * direction).sum(), rtol=1e-7, atol=1e-8)
    torch.testing.assert_close(along(lambda t: ref.layer_norm(x, gamma + t * v, beta, 1e-3)), (dgamma * v).sum(), rtol=1e-7, atol=1e-8)
    torch.testing.assert_close(along(lambda t: ref.layer_norm(x, gamma, beta + t * v, 1e-3)), (dbeta * v).sum(), rtol=1e-7, atol=1e-8)
    for value, slope in ref.ACTIVATIONS.values():
        torch.testing.assert_close((value(x + h) - value(x - h)) / (2 * h), slope(x), rtol=1e-7, atol=1e-8)


def test_the_definition_of_eight_bits():
    x = torch.tensor([[127.0, 0.5, 1.5, -2.5, 126.5, -127.0], [0.0, 0, 0, 0, 0, 0]])
    q, s = ref.int8(x)
    assert q.tolist() == [[127, 0, 2, -2, 126, -127], [0] * 6] and s[0].item() == 1.0
    y = torch.randn(4, 300)
    q, s = ref.int8(y)
    assert (q.abs().amax(-1) == 127).all()
    assert ((q * s - y.double()).abs() <= s * (0.5 + 2.0 ** -16)).all()
