"""A norm call that leaves a part out refuses that part's parameters, in both
directions: on the CPU, before any check of devices, and through the C ABI with
addresses that are never read."""

import pytest
import torch

import rollfast_b200 as rf
from rollfast_b200 import _lib

V = torch.ones(40)


@pytest.mark.parametrize("name", ["post_weight", "post_bias", "gate", "residual_scale"])
def test_parameters_of_an_absent_branch_are_refused(monkeypatch, name):
    import rollfast_b200.block_norm as bn

    monkeypatch.setattr(bn, "require_cuda", lambda t, what: None)
    x = torch.zeros(4, 40)
    with pytest.raises(ValueError, match=f"{name} given without a branch"):
        rf.block_norm_forward(x, **{name: V})
    with pytest.raises(ValueError, match=f"{name} given without a branch"):
        rf.block_norm_backward(x, x, x, **{name: V})


@pytest.mark.parametrize("name", ["pre_weight", "pre_bias"])
def test_parameters_of_an_absent_norm_are_refused(monkeypatch, name):
    import rollfast_b200.block_norm as bn

    monkeypatch.setattr(bn, "require_cuda", lambda t, what: None)
    x = torch.zeros(4, 40)
    with pytest.raises(ValueError, match=f"{name} given with pre_norm=False"):
        rf.block_norm_forward(x, x, pre_norm=False, **{name: V})


def test_c_abi_refuses_them_too():
    lib = _lib.load()

    def norm(name):
        p = _lib.RfBlockNorm(rows=4, features=40, kind=0, post_norm=1, eps=1e-6, scale=1.0, gate_rows=4)
        f = getattr(p, name)
        f.value, f.dtype = 4096, _lib.RF_F32
        return p

    a = _lib.RfRows(4096, 40, 1, None)
    for name in ("post_weight", "post_bias", "gate", "residual_scale"):
        assert lib.rf_block_norm_forward(norm(name), a, None, None, a, None, None, None, None) == _lib.RF_EINVAL
        assert b"without a branch" in lib.rf_last_error()
    for name in ("pre_weight", "pre_bias"):
        assert lib.rf_block_norm_forward(norm(name), a, a, a, None, None, None, None, None) == _lib.RF_EINVAL
        assert b"without y" in lib.rf_last_error()


@pytest.mark.gpu
def test_a_number_is_no_parameter_of_the_branch():
    x = torch.randn(4, 40, device="cuda")
    assert torch.equal(rf.block_norm_forward(x, residual_scale=0.5).y, rf.block_norm_forward(x).y)
