"""Arrays with more rows than the resident blocks of a kernel take in one
turn: noise, prefetched rows, steps and outputs from the second turn on."""

import numpy as np
import pytest
import torch

from oracle import training_np as T

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
# A turn is at most 148 SMs x 3 blocks x 256 threads x 4 rows of 8 features each: 3.6 million elements.
SHAPES = [(15_001, 256), (3_701, 1000), (2_001, 2312), (15_001, 264)]


def _rand(shape, dt, seed, scale=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dt)


def _same(a, b, rows):
    assert torch.equal(a.codes, torch.cat([s.codes for s in b]))
    assert torch.equal(a.scales[:, :rows], torch.cat([s.scales[:, :s.rows] for s in b], 1))


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("seed", [None, 12345])
def test_save_and_load(shape, dt, fmt, seed):
    import rollfast_b200 as rf

    x = _rand(shape, dt, 1)
    saved = rf.save_activation(x, fmt, seed=seed)
    codes, scales = T.encode8(x.float().cpu().numpy(), fmt, seed)
    assert np.array_equal(saved.codes.cpu().numpy(), codes)
    assert np.array_equal(saved.scales.cpu().numpy()[:, :shape[0]], scales[:, :shape[0]])
    want = torch.from_numpy(T.decode8(codes, scales, shape[1], fmt))
    for out in TYPES:
        assert torch.equal(rf.load_activation(saved, dtype=out).cpu(), want.to(out))


@pytest.mark.parametrize("shape", [*SHAPES, (9_001, 771)], ids=str)
@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_swiglu(shape, dt, fmt):
    """Rows are independent: the same bits as in calls of 1000 rows."""
    import rollfast_b200 as rf

    rows, d = shape
    both, dh = _rand((rows, 2 * d), dt, 2, 2.0), _rand(shape, dt, 3)
    gate, up = both[:, :d], both[:, d:]
    cuts = [slice(a, min(a + 1000, rows)) for a in range(0, rows, 1000)]
    h, sg, su = rf.swiglu_forward(gate, up, fmt)
    parts = [rf.swiglu_forward(gate[c], up[c], fmt) for c in cuts]
    assert torch.equal(h, torch.cat([p[0] for p in parts]))
    assert torch.equal(h, rf.swiglu_forward(gate, up, None)[0])
    _same(sg, [p[1] for p in parts], rows)
    _same(su, [p[2] for p in parts], rows)
    for save in (fmt, None):
        dg, du, sh = rf.swiglu_backward(dh, sg, su, save_h=save)
        back = [rf.swiglu_backward(dh[c], p[1], p[2], save_h=save) for c, p in zip(cuts, parts)]
        assert torch.equal(dg, torch.cat([p[0] for p in back])) and torch.equal(du, torch.cat([p[1] for p in back]))
        if save:
            _same(sh, [p[2] for p in back], rows)


@pytest.mark.parametrize("shape", [(20_000, 64), (5_001, 768), (2_003, 1001), (1_001, 5120), (701, 8200)], ids=str)
@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("gate", ["channel", "token"])
def test_block_norms(shape, dt, kind, gate):
    """Rows' outputs are independent of the other rows, and parameters' sums
    equal the sums of parts."""
    import rollfast_b200 as rf

    rows, d = shape
    x, b, dx, dy = (_rand(shape, dt, s) for s in (4, 5, 6, 7))
    p = {"pre_weight": _rand((d,), torch.float32, 8), "post_weight": _rand((d,), torch.float32, 9),
         "residual_scale": _rand((d,), torch.float32, 10)}
    gates = _rand((d,) if gate == "channel" else (rows, 1), torch.float32, 11)
    kw = dict(kind=kind, gate_activation="sigmoid")
    cuts = [slice(a, min(a + 97, rows)) for a in range(0, rows, 97)]

    def at(c):
        return gates if gate == "channel" else gates[c]

    r = rf.block_norm_forward(x, b, **p, gate=gates, save="int8", **kw)
    parts = [rf.block_norm_forward(x[c], b[c], **p, gate=at(c), save="int8", **kw) for c in cuts]
    assert torch.equal(r.x, torch.cat([q.x for q in parts])) and torch.equal(r.y, torch.cat([q.y for q in parts]))
    for name in ("saved_x", "saved_branch", "saved_y"):
        _same(getattr(r, name), [getattr(q, name) for q in parts], rows)
    for xs, bs, small in ((r.x, b, [(r.x[c], b[c]) for c in cuts]),
                          (r.saved_x, r.saved_branch, [(q.saved_x, q.saved_branch) for q in parts])):
        g = rf.block_norm_backward(dx, dy, xs, bs, **p, gate=gates, **kw)
        back = [rf.block_norm_backward(dx[c], dy[c], *s, **p, gate=at(c), **kw) for c, s in zip(cuts, small)]
        assert torch.equal(g.x, torch.cat([q.x for q in back])) and torch.equal(g.branch, torch.cat([q.branch for q in back]))
        for name in p:
            sums = [getattr(q, name).double() for q in back]
            # Float32 sums of n rows in any order: each within n U of its terms'
            # magnitudes, which no part's sum exceeds by more than its cancellation;
            # 20000 rows of about unit size: sqrt(rows) U a row.
            err = (getattr(g, name).double() - sum(sums)).abs().max()
            assert err <= rows * 2.0 ** -24 * 2 * max(1.0, float(sum(s.abs() for s in sums).max())), name
        if gate == "token":
            assert torch.equal(g.gate, torch.cat([q.gate for q in back]))


def test_one_row_at_a_time_of_a_wide_array():
    import rollfast_b200 as rf

    x = _rand((3, 28_672), torch.bfloat16, 12)
    whole = rf.save_activation(x, "e4m3")
    for i in range(3):
        one = rf.save_activation(x[i:i + 1], "e4m3")
        assert torch.equal(one.codes[0], whole.codes[i]) and torch.equal(one.scales[:, 0], whole.scales[:, i])
