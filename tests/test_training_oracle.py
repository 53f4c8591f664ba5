"""The 64-bit plain forms of the training-step operators against what defines
them: error bounds and minimality of the 8-bit form, unbiased stochastic
rounding, and every gradient against differences of its forward form."""

import numpy as np
import pytest

from oracle import training_np as T

FORMATS = ["int8", "e4m3"]


def _steps(scales, rows, features):
    s = scales[:, :rows].transpose(1, 0, 2).reshape(rows, -1).astype(int)
    return np.repeat(2.0 ** (s - 127.0), 32, axis=1)[:, :features]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", [(1, 1), (3, 33), (65, 130), (2, 768)])
def test_nearest_code_is_within_half_a_grid_step(fmt, shape):
    x = (np.random.default_rng(0).standard_normal(shape) * 3).astype(np.float32)
    codes, scales = T.encode8(x, fmt)
    v = T.decode8(codes, scales, shape[1], fmt)
    step = _steps(scales, *shape)
    if fmt == "int8":
        bound = step / 2
    else:  # half a unit in the fourth significant bit, 2^-10 steps below 2^-6
        bound = np.maximum(np.abs(x) * 2.0 ** -4, step * 2.0 ** -10)
    assert (np.abs(v - x) <= bound).all()
    # The step is the smallest that holds the block's largest magnitude.
    most = T.FORMATS[fmt][0]
    pad = np.zeros((shape[0], -(-shape[1] // 32) * 32))
    pad[:, :shape[1]] = np.abs(x)
    a = pad.reshape(shape[0], -1, 32).max(-1)
    s = step[:, ::32]
    assert (a <= most * s).all() and ((a > most * s / 2) | (s == 2.0 ** -126)).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_stochastic_codes_are_neighbours_and_unbiased(fmt):
    rng = np.random.default_rng(1)
    row = (rng.standard_normal(64)).astype(np.float32)
    n = 4096
    codes, scales = T.encode8(np.tile(row, (n, 1)), fmt, seed=12345)
    v = T.decode8(codes, scales, 64, fmt)
    step = _steps(scales, 1, 64)[0]
    if fmt == "e4m3":
        step = step * 2.0 ** (np.maximum(np.floor(np.log2(np.abs(row) / step)), -6) - 3)
    assert (np.abs(v - row) <= step).all()
    # The mean of n roundings: its standard deviation is at most step / (2 sqrt n);
    # the 16-bit noise adds at most 2^-16 of a step.  Six deviations.
    assert (np.abs(v.mean(0) - row) <= step * (6 / (2 * np.sqrt(n)) + 2.0 ** -16)).all()


def test_special_blocks():
    x = np.zeros((4, 64), np.float32)
    x[1, 3] = np.inf
    x[2, 40] = np.nan
    x[3] = 3.4e38
    for fmt in FORMATS:
        codes, scales = T.encode8(x, fmt)
        v = T.decode8(codes, scales, 64, fmt)
        assert (v[0] == 0).all() and scales[0, 0, 0] == 1
        assert np.isnan(v[1, :32]).all() and (v[1, 32:] == 0).all()
        assert np.isnan(v[2, 32:]).all() and (v[2, :32] == 0).all()
        assert np.isfinite(v[3].astype(np.float32)).all()
        assert (v[3] == T.FORMATS[fmt][0] * 2.0 ** (T.FORMATS[fmt][1] - 127)).all()


def _difference(f, v, h=1e-6):
    g = np.zeros_like(v)
    for i in np.ndindex(*v.shape):
        a, b = v.copy(), v.copy()
        a[i] += h
        b[i] -= h
        g[i] = (f(a) - f(b)) / (2 * h)
    return g


def test_swiglu_gradients_against_differences():
    rng = np.random.default_rng(2)
    g, u, d = rng.standard_normal((3, 5, 7)) * 2
    dg, du = T.swiglu_grads(d, g, u)
    assert np.allclose(dg, _difference(lambda v: (d * T.swiglu(v, u)).sum(), g), atol=1e-7)
    assert np.allclose(du, _difference(lambda v: (d * T.swiglu(g, v)).sum(), u), atol=1e-7)


def test_weight_gradient_against_differences():
    rng = np.random.default_rng(3)
    x, g, w = rng.standard_normal((2, 3, 4)), rng.standard_normal((2, 3, 5)), rng.standard_normal((4, 5))
    want = _difference(lambda v: ((x @ v) * g).sum(), w)
    assert np.allclose(T.weight_gradient(x, g), want, atol=1e-7)
    assert np.allclose(T.weight_gradient(x, g, initial=w.T, layout="oi"), want.T + w.T, atol=1e-7)


GATES = {"none": None, "channel": (6,), "sequence": (2, 1, 6), "token": (2, 3, 1), "full": (2, 3, 6), "one": (1,)}


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("post_norm", [True, False])
@pytest.mark.parametrize("gate", list(GATES))
@pytest.mark.parametrize("act", [None, "sigmoid", "tanh"])
@pytest.mark.parametrize("scale", [None, 0.3, (6,), (1,)])
def test_block_norm_gradients_against_differences(kind, post_norm, gate, act, scale):
    rng = np.random.default_rng(4)
    shape = (2, 3, 6)
    x, b, dx, dy = rng.standard_normal((4, *shape))
    p = {"pre_weight": rng.standard_normal(6), "pre_bias": rng.standard_normal(6)}
    if post_norm:
        p |= {"post_weight": rng.standard_normal(6), "post_bias": rng.standard_normal(6)}
    if GATES[gate]:
        p["gate"] = rng.standard_normal(GATES[gate])
    if scale is not None:
        p["residual_scale"] = rng.standard_normal(scale) if isinstance(scale, tuple) else scale
    kw = dict(kind=kind, eps=1e-3, post_norm=post_norm, gate_activation=act)

    def loss(x, b, p):
        out, y = T.block_norm(x, b, p, **kw)
        return (out * dx).sum() + (y * dy).sum()

    got = T.block_norm_grads(dx, dy, T.block_norm(x, b, p, **kw)[0], b, p, **kw)
    assert np.allclose(got["x"], _difference(lambda v: loss(v, b, p), x), atol=1e-6)
    assert np.allclose(got["branch"], _difference(lambda v: loss(x, v, p), b), atol=1e-6)
    for name, v in p.items():
        if np.ndim(v):
            assert got[name].shape == np.shape(v)
            assert np.allclose(got[name], _difference(lambda q: loss(x, b, p | {name: q}), v), atol=1e-6), name
