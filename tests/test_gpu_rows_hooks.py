"""Layer normalisation's backward pass where a hook brings back an input that is not the one that was saved, the statistics
as they were."""
import pytest
import torch

from approxtrain_amd import math_ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("other", [lambda t: t[:0], lambda t: t[:-1], lambda t: t[:, :-1], lambda t: t.t(), lambda t: t.double(), lambda t: t.cpu(), lambda t: t[None],
                                   lambda t: t.to_sparse()],
                         ids=["no rows", "fewer rows", "fewer columns", "transposed", "64 bits", "on the host", "an axis more", "sparse"])
def test_another_input_is_refused(other):
    x = torch.randn(20, 64, device="cuda", requires_grad=True)
    gamma = torch.ones(64, device="cuda", requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: other(t) if t.shape == (20, 64) else t):
        y = math_ops.layernorm(x, gamma)
    with pytest.raises(RuntimeError, match="layernorm kept for its backward pass came back in another form"):
        y.sum().backward()


def test_the_same_values_in_other_strides_are_not():
    x = torch.randn(20, 64, device="cuda", requires_grad=True)
    dy = torch.randn(20, 64, device="cuda")
    want, = torch.autograd.grad(math_ops.layernorm(x), [x], dy)
    for other in (lambda t: t.t().contiguous().t(), lambda t: torch.stack([t, t], -1)[..., 0]):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: other(t) if t.shape == (20, 64) else t):
            y = math_ops.layernorm(x)
        assert torch.equal(torch.autograd.grad(y, [x], dy)[0], want)
