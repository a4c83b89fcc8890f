"""The packed layer's saved state, on the host: the conversion is replaced by one that makes empty operands."""
import pytest
import torch

from approxtrain_amd import functors, load_library
from approxtrain_amd.layers import packed_densemx
from approxtrain_amd.mx import MXTensor


@pytest.fixture(autouse=True)
def host_conversion(monkeypatch):
    def quantize(x, axis):
        assert axis == 0
        n = load_library().amsim_mxfp4_operand_workspace_bytes(x.shape[1], x.shape[0])
        return MXTensor(torch.zeros(n, dtype=torch.uint8), x.shape[1], x.shape[0])
    monkeypatch.setattr(functors, "mxfp4_quantize", quantize)


def packed(width, units, byte=0):
    layer = packed_densemx(torch.zeros(width, units), torch.zeros(units), "relu")
    layer.weights.fill_(byte)
    return layer


def test_weights_of_other_extents_do_not_load():
    """Operands of 70 and of 100 values a row take as many bytes."""
    source = torch.nn.Sequential(packed(100, 33, 7))
    for width, units in ((70, 33), (100, 34)):
        target = torch.nn.Sequential(packed(width, units))
        if units == 33:
            assert target[0].weights.shape == source[0].weights.shape
        with pytest.raises(RuntimeError, match="100"):
            target.load_state_dict(source.state_dict())
        assert not target[0].weights.any()
    target = torch.nn.Sequential(packed(100, 33))
    target.load_state_dict(source.state_dict())
    assert bool((target[0].weights == 7).all())


def test_states_saved_without_extents_load():
    source = torch.nn.Sequential(packed(100, 33, 7)).state_dict()
    old = {k: v for k, v in source.items() if k in ("0.weights", "0.bias")}
    target = torch.nn.Sequential(packed(100, 33))
    target.load_state_dict(old)
    assert bool((target[0].weights == 7).all())
    for k in list(source):
        if k not in old:
            del source[k]
    with pytest.raises(RuntimeError, match="Missing"):
        torch.nn.Sequential(packed(100, 33)).load_state_dict(source)
