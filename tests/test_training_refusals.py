"""Refusals of the training-step operators, on the CPU: what reaches no
kernel -- Python's checks, and the C ABI's with addresses that are never read."""

import ctypes

import pytest
import torch

import rollfast_b200 as rf
from rollfast_b200 import _lib
from rollfast_b200.activations import row_strided
from rollfast_b200.block_norm import _gate_layout


def _saved(rows=4, d=40, fmt="int8", shape=None):
    return rf.SavedActivation(torch.zeros(rows, -(-d // 16) * 16, dtype=torch.uint8),
                              torch.ones(-(-d // 128), -(-rows // 64) * 64, 4, dtype=torch.uint8),
                              shape or (rows, d), torch.bfloat16, fmt)


def test_saved_activation_checks_its_layout():
    s = _saved(shape=(2, 2, 40))
    assert (s.rows, s.features, s.shape) == (4, 40, (2, 2, 40)) and s.nbytes == 4 * 48 + 256
    c, sc = s.codes, s.scales
    for bad in [
        lambda: rf.SavedActivation(c[:, :40], sc, (4, 40), torch.bfloat16, "int8"),
        lambda: rf.SavedActivation(c, sc[:, :4], (4, 40), torch.bfloat16, "int8"),
        lambda: rf.SavedActivation(c.to(torch.int8), sc, (4, 40), torch.bfloat16, "int8"),
        lambda: rf.SavedActivation(c, sc, (5, 40), torch.bfloat16, "int8"),
        lambda: rf.SavedActivation(c, sc, (4, 40), torch.bfloat16, "e5m2"),
        lambda: rf.SavedActivation(c, sc, (), torch.bfloat16, "int8"),
        lambda: rf.SavedActivation(c, sc, (4, 0), torch.bfloat16, "int8"),
    ]:
        with pytest.raises(ValueError):
            bad()


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 40)
    s = _saved()
    for call in [
        lambda: rf.save_activation(x),
        lambda: rf.load_activation(s),
        lambda: rf.load_activation(x),
        lambda: rf.weight_gradient(s, x),
        lambda: rf.weight_gradient(x, x),
        lambda: rf.swiglu_forward(x, x),
        lambda: rf.swiglu_backward(x, s, s),
        lambda: rf.block_norm_forward(x),
        lambda: rf.block_norm_forward(x, x),
        lambda: rf.block_norm_backward(x, x, x),
        lambda: rf.block_norm_backward(x, x, s, s),
        lambda: rf.block_norm_backward(None, None, x),
    ]:
        with pytest.raises(ValueError):
            call()


def test_gate_layouts():
    shape = (2, 3, 5, 8)
    assert _gate_layout((8,), shape) == (30, True)
    assert _gate_layout((1,), shape) == (30, False)
    assert _gate_layout((), shape) == (30, False)
    assert _gate_layout((2, 1, 1, 8), shape) == (15, True)
    assert _gate_layout((2, 3, 1, 1), shape) == (5, False)
    assert _gate_layout((2, 3, 5, 1), shape) == (1, False)
    assert _gate_layout(shape, shape) == (1, True)
    assert _gate_layout((8,), (0, 8)) == (1, True)
    for bad in [(3, 5, 8), (1, 3, 1, 8), (1, 1, 5, 8), (2, 3, 4, 8), (7,), (2, 2, 3, 5, 8)]:
        with pytest.raises(ValueError):
            _gate_layout(bad, shape)


def test_row_strides():
    x = torch.zeros(4, 6, 20)
    for view, ld in [(x, 20), (x[..., 3:9], 20), (x[:, 0], 120), (x[0], 20), (x[:, :1, 2:5], 120), (x[0, 0], 20)]:
        same, got = row_strided(view)
        assert same is view and got == ld
    for view in [x.transpose(0, 1)[..., :4], x[..., ::2], x[:, :3], x[:1].expand(4, 6, 20), x[:, 0, :1].expand(4, 5)]:
        same, got = row_strided(view)
        assert same is not view and same.is_contiguous() and got == view.shape[-1]


def _c_saved(rows=4, d=40, fmt=0, codes=1024, scales=2048, **other):
    s = _lib.RfSavedActivation(codes, scales, rows, d, -(-d // 16) * 16, -(-rows // 64) * 64, fmt)
    for k, v in other.items():
        setattr(s, k, v)
    return s


def _invalid(status):
    assert status == _lib.RF_EINVAL
    assert _lib.load().rf_last_error()


def test_c_abi_refuses_bad_saved_activations():
    lib = _lib.load()
    for s in [None, _c_saved(fmt=2), _c_saved(rows=-1), _c_saved(d=0), _c_saved(ld=40), _c_saved(scale_rows=4),
              _c_saved(codes=None), _c_saved(scales=2056), _c_saved(codes=1032), _c_saved(rows=1 << 31),
              _c_saved(d=(1 << 26) + 1)]:
        _invalid(lib.rf_save_activation(4096, 1 << 27, 1, s, 0, 0, None))
        _invalid(lib.rf_load_activation(s, 4096, 1 << 27, 1, None))
        _invalid(lib.rf_weight_gradient(s, 4096, 24, 1, 24, 0, None, 8192, 24, 0, None, 0, None))
        _invalid(lib.rf_swiglu_backward(4096, 1 << 27, s, s, 4096, 1 << 27, 4096, 1 << 27, 1, None, None))


def test_c_abi_refuses_bad_arrays():
    lib = _lib.load()
    s = _c_saved()
    _invalid(lib.rf_save_activation(None, 40, 1, s, 0, 0, None))
    _invalid(lib.rf_save_activation(4096, 39, 1, s, 0, 0, None))
    _invalid(lib.rf_save_activation(4097, 40, 1, s, 0, 0, None))
    _invalid(lib.rf_save_activation(4096, 40, 7, s, 0, 0, None))
    _invalid(lib.rf_load_activation(s, None, 40, 1, None))
    _invalid(lib.rf_swiglu_forward(4096, 40, 4096, 40, 4096, 40, 1, 4, 40, s, None, None))
    _invalid(lib.rf_swiglu_forward(4096, 40, 4096, 40, 4096, 40, 1, 5, 40, s, s, None))
    _invalid(lib.rf_swiglu_forward(4096, 40, 4096, 40, 4096, 40, 1, -1, 40, None, None, None))
    _invalid(lib.rf_swiglu_backward(4096, 40, s, _c_saved(rows=5), 4096, 40, 4096, 40, 1, None, None))
    _invalid(lib.rf_swiglu_backward(4096, 40, s, s, 4096, 40, 4096, 40, 1, _c_saved(d=41), None))


def test_c_abi_weight_gradient_plans_and_refuses():
    lib = _lib.load()
    n = ctypes.c_size_t()

    def plan(rows, k, out, ptr, ld, dt):
        _lib.check(lib.rf_weight_gradient_workspace_size(rows, k, out, ptr, ld, dt, ctypes.byref(n)))
        return n.value

    x, tile = 8192 * 4096 * 2, 256 * 256 * 4
    whole = plan(8192, 4096, 74 * 256, 4096, 74 * 256, _lib.RF_BF16)           # full waves of tiles, read in place
    assert whole == x                                                        # the expanded activation
    assert plan(8192, 4096, 74 * 256, 4098, 74 * 256, _lib.RF_BF16) == x + 8192 * 74 * 256 * 2   # misaligned: copied
    assert plan(8192, 4096, 74 * 256, 4096, 74 * 256, _lib.RF_F32) == x + 3 * 8192 * 74 * 256 * 2
    assert plan(0, 40, 24, None, 24, _lib.RF_F32) == 0
    split = plan(4096, 768, 768, 4096, 768, _lib.RF_BF16) - 4096 * 768 * 2
    assert split > 0 and split % (9 * tile) == 0                             # 9 tiles, each in parts
    _invalid(lib.rf_weight_gradient_workspace_size(4, 40, 24, None, 23, 1, ctypes.byref(n)))
    _invalid(lib.rf_weight_gradient_workspace_size(4, 40, 0, None, 24, 1, ctypes.byref(n)))
    _invalid(lib.rf_weight_gradient_workspace_size(4, 40, 24, None, 24, 9, ctypes.byref(n)))
    _invalid(lib.rf_weight_gradient_workspace_size(4, 40, 24, None, 24, 1, None))
    s = _c_saved()
    ok = [s, 4096, 24, 1, 24, 0, None, 8192, 24, 0, None, 0, None]
    for i, v in [(1, None), (2, 20), (3, 5), (4, 0), (5, 2), (7, None), (8, 23), (9, 4), (1, 4097), (7, 8193), (6, 8194)]:
        bad = list(ok)
        bad[i] = v
        _invalid(lib.rf_weight_gradient(*bad))
    need = list(ok)  # the expanded activation needs a workspace
    _invalid(lib.rf_weight_gradient(*need))
    need[10], need[11] = 4097, 1 << 20
    _invalid(lib.rf_weight_gradient(*need))


def test_c_abi_block_norm_refuses():
    lib = _lib.load()

    def norm(**kw):
        p = _lib.RfBlockNorm(rows=4, features=40, kind=0, post_norm=1, eps=1e-6, scale=1.0, gate_rows=1)
        for k, v in kw.items():
            if isinstance(v, tuple):
                f = getattr(p, k)
                f.value, f.grad, f.dtype = v
            else:
                setattr(p, k, v)
        return p

    a = _lib.RfRows(4096, 40, 1, None)
    for p in [norm(rows=-1), norm(features=0), norm(features=16385), norm(kind=2), norm(eps=-1.0), norm(eps=float("nan")),
              norm(pre_weight=(4096, None, 9)), norm(pre_weight=(4097, None, 1)), norm(pre_weight=(None, 4096, 1)),
              norm(post_norm=0, post_weight=(4096, None, 1)), norm(gate=(4096, None, 1), gate_rows=3),
              norm(gate=(4096, None, 1), gate_rows=0), norm(gate=(4096, None, 1), gate_act=3)]:
        _invalid(lib.rf_block_norm_forward(p, a, a, a, a, None, None, None, None))
        _invalid(lib.rf_block_norm_backward(p, a, a, a, a, a, a, 4096, 1 << 20, None))
        _invalid(lib.rf_block_norm_workspace_size(p, ctypes.byref(ctypes.c_size_t())))
    s = _c_saved()
    p = norm()
    bad = [_lib.RfRows(None, 40, 1, None), _lib.RfRows(4096, 39, 1, None), _lib.RfRows(4097, 40, 1, None),
           _lib.RfRows(4096, 40, 8, None), _lib.RfRows(None, 0, 0, ctypes.pointer(s))]
    for b in bad:
        _invalid(lib.rf_block_norm_forward(p, b, a, a, a, None, None, None, None))
    for b in bad[1:]:
        _invalid(lib.rf_block_norm_forward(p, a, b, a, a, None, None, None, None))
        _invalid(lib.rf_block_norm_backward(p, b, a, a, a, a, a, None, 0, None))
    _invalid(lib.rf_block_norm_forward(None, a, a, a, a, None, None, None, None))
    _invalid(lib.rf_block_norm_forward(p, a, a, None, a, None, None, None, None))
    _invalid(lib.rf_block_norm_forward(p, a, None, None, a, None, s, None, None))
    _invalid(lib.rf_block_norm_forward(p, a, a, a, None, None, None, s, None))
    _invalid(lib.rf_block_norm_forward(p, a, a, a, a, _c_saved(rows=5), None, None, None))
    wants = norm(pre_weight=(4096, 8192, 1))
    _invalid(lib.rf_block_norm_backward(wants, a, a, a, a, a, a, None, 0, None))
    _invalid(lib.rf_block_norm_backward(wants, a, a, a, a, a, a, 4097, 1 << 20, None))
    _invalid(lib.rf_block_norm_backward(norm(gate=(4096, 8192, 1)), a, a, a, None, a, None, 4096, 1 << 20, None))


def test_calls_without_rows_launch_nothing():
    lib = _lib.load()
    before = _lib.kernel_launch_count()
    s = _c_saved(rows=0, codes=None, scales=None)
    _lib.check(lib.rf_save_activation(None, 40, 1, s, 0, 0, None))
    _lib.check(lib.rf_load_activation(s, None, 40, 1, None))
    _lib.check(lib.rf_swiglu_forward(None, 40, None, 40, None, 40, 1, 0, 40, s, s, None))
    _lib.check(lib.rf_swiglu_backward(None, 40, s, s, None, 40, None, 40, 1, s, None))
    assert _lib.kernel_launch_count() == before
