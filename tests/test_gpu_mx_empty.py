"""Batches of no rows, as a router may leave to an expert: empty results, and gradients of zeros."""
import pytest
import torch

from approxtrain_amd import functors, math_ops
from approxtrain_amd.layers import densemx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(0, 40), (2, 0, 40), (0, 3, 40)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("activation", [None, "relu"])
def test_no_rows(shape, dtype, activation):
    x = torch.zeros(shape, device="cuda", dtype=dtype, requires_grad=True)
    w, b = torch.randn(40, 24, device="cuda", requires_grad=True), torch.randn(24, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    out = math_ops.linearmx(x, w, b, activation)
    assert out.shape == shape[:-1] + (24,) and out.dtype == dtype
    gx, gw, gb = torch.autograd.grad(out.sum(), [x, w, b])
    assert gx.shape == shape and gx.dtype == dtype
    assert torch.equal(gw, torch.zeros_like(w)) and torch.equal(gb, torch.zeros_like(b))
    gw, = torch.autograd.grad(math_ops.linearmx(x.detach(), w, b, activation).sum(), [w])
    assert torch.equal(gw, torch.zeros_like(w))
    with torch.no_grad():
        assert math_ops.linearmx(x, w, b, activation).shape == out.shape


def test_layers_and_calls_of_no_rows():
    layer = densemx(24, "tanh", input_dim=40).cuda()
    layer(torch.zeros(0, 40, device="cuda")).sum().backward()
    assert not layer.kernel.grad.any() and not layer.bias.grad.any()
    assert layer.pack()(torch.zeros(0, 40, device="cuda")).shape == (0, 24)
    x, w = torch.zeros(0, 40, device="cuda"), torch.randn(40, 24, device="cuda")
    out, kept = functors.mxfp4_dense(x, w)
    assert out.shape == (0, 24)
    grads = functors.mxfp4_dense_grad(out, kept, 0, 40, 24, kernel_dtype=torch.float32, bias_dtype=torch.float32)
    assert [tuple(g.shape) for g in grads] == [(0, 40), (40, 24), (24,)] and not grads[1].any() and not grads[2].any()


def test_refusals():
    w = torch.randn(40, 24, device="cuda")
    with pytest.raises(ValueError, match="no elements"):
        math_ops.linearmx(torch.zeros(5, 0, device="cuda"), torch.zeros(0, 24, device="cuda"))
    with pytest.raises(ValueError, match="no elements"):
        math_ops.linearmx(torch.zeros(0, 40, device="cuda"), torch.zeros(40, 0, device="cuda"))
    with pytest.raises(TypeError, match="x must be"):
        math_ops.linearmx(torch.zeros(0, 40, device="cuda", dtype=torch.float64), w)
    with pytest.raises(ValueError, match="bias"):
        math_ops.linearmx(torch.zeros(0, 40, device="cuda"), w, torch.zeros(23, device="cuda"))
    with pytest.raises(TypeError, match="device memory"):
        math_ops.linearmx(torch.zeros(0, 40), w)
    with pytest.raises(ValueError, match="shape"):
        functors.mxfp4_dense_grad(torch.zeros(1, 24, device="cuda"), torch.zeros(0, dtype=torch.uint8, device="cuda"), 0, 40, 24)
