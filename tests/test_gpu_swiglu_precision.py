"""Float32 SwiGLU is as exact where the gate is strongly negative as elsewhere.

Bounds, in U = 2^-24 relative, to first order (the factor 1.01 covers the
rest).  exp(-|g|) is off by at most two units of float32, 4 U.  In
s = e / (1 + e) or 1 / (1 + e), e's error enters with a weight of at most 1,
the sum and the quotient are rounded once each: 6 U.  h = g s u: two roundings
more, 8 U.  du = d (g s): 8 U too.  The slope s + a (1 - s), a = g s (7 U): with
1 - s off by 6 U s and U of itself, and two roundings of the whole,
    s 6 U + |a| (1 - s) (7 + 1) U + |a| s 6 U + 2 U (s + |a| (1 - s))
        <= s (1 + |g|) 16 U,
and dg = (d u) slope two roundings more: 18 U."""

import numpy as np
import pytest
import torch

from oracle import training_np as T

pytestmark = pytest.mark.gpu

U = 2.0 ** -24 * 1.01
TINY = 2.0 ** -148


def _np(t):
    return t.detach().to(torch.float64).cpu().numpy()


def _gates(rows, d, seed):
    rng = np.random.default_rng(seed)
    return torch.from_numpy(rng.uniform(-80.0, 80.0, (rows, d)).astype(np.float32)).cuda()


@pytest.mark.parametrize("d", [256, 257])
def test_float32_forward(d):
    import rollfast_b200 as rf

    g, u = _gates(301, d, 1), torch.randn(301, d, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    want = T.swiglu(_np(g), _np(u))
    for fmt in ("int8", None):
        h = rf.swiglu_forward(g, u, fmt)[0]
        assert (np.abs(_np(h) - want) <= np.abs(want) * 8 * U + TINY).all()


@pytest.mark.parametrize("d", [256, 257])
@pytest.mark.parametrize("save", [None, "e4m3"])
def test_float32_backward(d, save):
    import rollfast_b200 as rf

    gen = torch.Generator("cuda").manual_seed(3)
    u, dh = (torch.randn(301, d, device="cuda", generator=gen) for _ in range(2))
    _, sg, su = rf.swiglu_forward(_gates(301, d, 4), u, "int8")
    dg, du, _ = rf.swiglu_backward(dh, sg, su, save_h=save)
    g, v, e = (_np(t) for t in (rf.load_activation(sg), rf.load_activation(su), dh))
    wg, wu = T.swiglu_grads(e, g, v)
    s = 1 / (1 + np.exp(-g))
    assert (np.abs(_np(du) - wu) <= np.abs(wu) * 8 * U + TINY).all()
    assert (np.abs(_np(dg) - wg) <= np.abs(e * v) * s * (1 + np.abs(g)) * 18 * U + TINY).all()
