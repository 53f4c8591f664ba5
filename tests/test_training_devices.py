"""Arrays of one call on two devices are refused before any launch.  Meta
tensors stand for another GPU's: the checks compare devices, whichever."""

import pytest
import torch

import rollfast_b200 as rf
import rollfast_b200.activations as act
import rollfast_b200.block_norm as bn


@pytest.fixture(autouse=True)
def any_device_is_a_gpu(monkeypatch):
    for module in (act, bn):
        monkeypatch.setattr(module, "require_cuda", lambda t, what: None)


def _saved(device):
    return rf.SavedActivation(torch.zeros(4, 48, dtype=torch.uint8, device=device),
                              torch.ones(1, 64, 4, dtype=torch.uint8, device=device), (4, 40), torch.bfloat16, "int8")


def _array(device, *shape):
    return torch.zeros(*(shape or (4, 40)), dtype=torch.bfloat16, device=device)


@pytest.mark.parametrize("call", [
    lambda a, b: rf.weight_gradient(_saved(a), _array(b)),
    lambda a, b: rf.weight_gradient(_saved(a), _array(a), initial=_array(b, 40, 40)),
    lambda a, b: rf.weight_gradient(_saved(a), _array(a), out=_array(b, 40, 40)),
    lambda a, b: rf.swiglu_forward(_array(a), _array(b)),
    lambda a, b: rf.swiglu_backward(_array(a), _saved(b), _saved(a)),
    lambda a, b: rf.swiglu_backward(_array(a), _saved(a), _saved(b)),
    lambda a, b: rf.swiglu_backward(_array(a), _saved(a), _saved(a), grad_up=_array(b)),
    lambda a, b: rf.block_norm_forward(_array(a), _array(b)),
    lambda a, b: rf.block_norm_forward(_array(a), pre_weight=_array(b, 40)),
    lambda a, b: rf.block_norm_forward(_array(a), _array(a), gate=_array(b, 40)),
    lambda a, b: rf.block_norm_backward(_array(b), None, _array(a)),
    lambda a, b: rf.block_norm_backward(None, _array(b), _saved(a)),
    lambda a, b: rf.block_norm_backward(_array(a), None, _array(a), _saved(b)),
    lambda a, b: rf.block_norm_backward(_array(a), None, _array(a), pre_weight=_array(b, 40)),
])
@pytest.mark.parametrize("pair", [("cpu", "meta"), ("meta", "cpu")])
def test_two_devices_are_refused(call, pair):
    with pytest.raises(ValueError, match="is on .*, expected"):
        call(*pair)


def test_a_saved_activation_lies_on_one_device():
    s = _saved("cpu")
    with pytest.raises(ValueError, match="one device"):
        rf.SavedActivation(s.codes, s.scales.to("meta"), s.shape, s.dtype, s.format)
