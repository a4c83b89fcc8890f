"""LayerNormalization's arguments: those of every other layer here, and the last axis by its index."""
import pytest
import torch

from approxtrain_amd import functors, layers


def test_what_every_layer_takes():
    layer = layers.LayerNormalization(name="norm", trainable=False, dtype="float32", input_shape=(7, 40), gamma_regularizer=lambda t: t.sum(),
                                      beta_regularizer=lambda t: t.sum() + 1, gamma_constraint=lambda t: t * 2, beta_constraint=lambda t: t - 1)
    assert layer.layer_name == "norm" and layer.gamma.shape == layer.beta.shape == (40,) and not any(p.requires_grad for p in layer.parameters())
    assert [float(v) for v in layer.losses()] == [40.0, 1.0]
    layer.apply_constraints()
    assert (layer.gamma == 2).all() and (layer.beta == -1).all()
    bare = layers.LayerNormalization(center=False, scale=False, gamma_regularizer=lambda t: t.sum(), gamma_constraint=lambda t: t, input_dim=4)
    bare.apply_constraints()
    assert bare.losses() == []


@pytest.mark.parametrize("bad,error", [
    (dict(gamma_regularizer=1e-4), ValueError), (dict(beta_regularizer="l2"), ValueError), (dict(gamma_constraint=1), ValueError), (dict(beta_constraint=1), ValueError),
    (dict(dtype="float16"), ValueError), (dict(units=3), TypeError), (dict(axis=(1, 2)), ValueError), (dict(axis=[]), ValueError), (dict(axis=0), ValueError),
    (dict(axis=-2), ValueError), (dict(axis=None), ValueError)])
def test_refusals(bad, error):
    with pytest.raises(error):
        layers.LayerNormalization(**bad)


@pytest.mark.parametrize("axis", [1, [1], 3])
def test_another_axis_than_the_last_is_refused(axis):
    with pytest.raises(ValueError, match="last axis"):
        layers.LayerNormalization(axis=axis)(torch.ones(2, 3, 4))


@pytest.mark.gpu
@pytest.mark.parametrize("axis", [-1, 2, [2], (-1,)])
def test_the_last_axis_by_its_index(axis):
    x = torch.randn(3, 5, 40, device="cuda", requires_grad=True)
    layer = layers.LayerNormalization(axis=axis, activity_regularizer=lambda t: t.square().mean())
    y = layer(x)
    assert torch.equal(y.detach(), functors.layer_norm(x.detach(), layer.gamma.detach(), layer.beta.detach()))
    loss, = layer.losses()
    loss.backward()
    assert layer.gamma.grad.shape == (40,) and x.grad.shape == x.shape
