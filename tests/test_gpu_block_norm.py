"""Block norms, forward and backward, against the 64-bit plain forms
(oracle/training_np.py).

Tolerances, by arithmetic.  A row's sums of d float32 terms are formed by
threads over at most 32 terms, then in a tree of at most 5 levels, then over
at most 16 warps, so each is off by at most K = 64 half units (U = 2^-24) of
the sum of its terms' magnitudes; a handful of further roundings are inside
the same K.  Each test scales K U by the magnitudes that enter a result, and
adds the output's half step, finfo.eps / 2 of the value."""

import itertools

import numpy as np
import pytest
import torch

from oracle import training_np as T

pytestmark = pytest.mark.gpu

TORCH = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
U = 2.0 ** -24
K = 64
EPS = 1e-5


def _np(t):
    return t.detach().to(torch.float64).cpu().numpy()


def _half(dt):
    return torch.finfo(dt).eps / 2


def _tiny(dt):
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps


def _make(shape, dt, seed, scale=1.0, mean=0.0):
    rng = np.random.default_rng(seed)
    return torch.from_numpy((rng.standard_normal(shape) * scale + mean).astype(np.float32)).cuda().to(TORCH[dt])


def _setup(shape, dt, kind, post_norm, gate, act, scale, affine=True, pdt="float32"):
    d = shape[-1]
    x, b = _make(shape, dt, 1, 2.0, 0.3), _make(shape, dt, 2, 0.7, -0.2)
    p = {}
    if affine:
        p["pre_weight"] = _make((d,), pdt, 3, 0.2, 1.0)
        if kind == "layer":
            p["pre_bias"] = _make((d,), pdt, 4, 0.2)
        if post_norm:
            p["post_weight"] = _make((d,), pdt, 5, 0.2, 1.0)
            if kind == "layer":
                p["post_bias"] = _make((d,), pdt, 6, 0.2)
    shapes = {"none": None, "channel": (d,), "sequence": (shape[0],) + (1,) * (len(shape) - 2) + (d,),
              "token": shape[:-1] + (1,), "full": shape, "one": (1,), "sequence_scalar": (shape[0],) + (1,) * (len(shape) - 1)}
    if shapes[gate]:
        p["gate"] = _make(shapes[gate], pdt, 7, 0.8)
    if scale == "vector":
        p["residual_scale"] = _make((d,), pdt, 8, 0.3, 0.5)
    elif scale == "one":
        p["residual_scale"] = _make((1,), pdt, 9, 0.3, 0.5)
    elif scale == "number":
        p["residual_scale"] = 0.35
    kw = dict(kind=kind, eps=EPS, post_norm=post_norm)
    return x, b, p, kw, {"gate_activation": act}


def _plain(p):
    return {k: _np(v) if isinstance(v, torch.Tensor) else v for k, v in p.items()}


def _near(got, want, slack, what):
    dt = got.dtype
    err = np.abs(_np(got) - want)
    bound = slack + np.abs(want) * _half(dt) + _tiny(dt)
    assert (err <= bound).all(), f"{what}: worst error over bound {np.max(err / bound):.3g}"


def _norm_error(v, kind):
    """Bound of the error of a normalised row, absolute: relative K U on the
    values and, for a mean taken off, K U of the row's mean magnitude, in units
    of the root."""
    n, r = T.normalised(v, kind, EPS)
    e = np.abs(n) * K * U
    if kind == "layer":
        e = e + (np.abs(v) + np.abs(v).mean(-1, keepdims=True)) * r * K * U
    return e


def _check_forward(x, b, p, kw, akw, save=None):
    import rollfast_b200 as rf

    r = rf.block_norm_forward(x, b, **kw, **akw, **p, save=save)
    q = _plain(p)
    wx, wy = T.block_norm(_np(x), _np(b), q, **kw, **akw)
    m = _norm_error(_np(b), kw["kind"]) if kw["post_norm"] else np.zeros_like(wx)
    w, s = q.get("post_weight", 1.0), np.abs(q.get("residual_scale", 1.0))
    a = np.abs(T.gate_act(q["gate"], akw["gate_activation"])) if "gate" in q else 1.0
    ex = (m * np.abs(w) + (np.abs(wx - _np(x)) / np.maximum(s * a, 1e-30)) * K * U) * s * a + np.abs(wx) * 2 * U
    _near(r.x, wx, ex, "x")
    # y: the error of x' enters through the normalisation: relative to the row,
    # at most twice its own share and its mean over the row.
    n, rr = T.normalised(wx, kw["kind"], EPS)
    ey = _norm_error(wx, kw["kind"]) + rr * (ex + np.abs(n) * (np.abs(n) * ex).mean(-1, keepdims=True)
                                             + ex.mean(-1, keepdims=True)) * 2
    _near(r.y, wy, ey * np.abs(q.get("pre_weight", 1.0)) + np.abs(q.get("pre_bias", 0.0)) * 4 * U + np.abs(wy) * 4 * U, "y")
    if save:
        for t, sv in ((r.x, r.saved_x), (b, r.saved_branch), (r.y, r.saved_y)):
            alone = rf.save_activation(t, save)
            assert sv.shape == tuple(t.shape) and sv.dtype == t.dtype and sv.format == save
            assert torch.equal(sv.codes, alone.codes) and torch.equal(sv.scales[:, :sv.rows], alone.scales[:, :sv.rows])
        bare = rf.block_norm_forward(x, b, **kw, **akw, **p)
        assert torch.equal(bare.x, r.x) and torch.equal(bare.y, r.y) and bare[2:] == (None, None, None)
    return r


def _check_backward(x, b, p, kw, akw, dx, dy, save=None):
    """x is x'."""
    import rollfast_b200 as rf

    xs, bs = x, b
    if save:
        xs, bs = rf.save_activation(x, save), rf.save_activation(b, save)
        x, b = rf.load_activation(xs, dtype=torch.float32), rf.load_activation(bs, dtype=torch.float32)
    r = rf.block_norm_backward(dx, dy, xs, bs, **kw, **akw, **p)
    q = _plain(p)
    gx, gy = (None if t is None else _np(t) for t in (dx, dy))
    want = T.block_norm_grads(gx, gy, _np(x), _np(b), q, **kw, **akw)
    kind = kw["kind"]
    lead = tuple(range(x.ndim - 1))
    zero = np.zeros(tuple(x.shape))
    gx, gy = (zero if g is None else g for g in (gx, gy))

    def back(g, eg, n, en, r_):
        """Error of (g - n mean(g n) - mean g) r for errors eg of g and en of n."""
        mag = np.abs(g) + np.abs(n) * (np.abs(g * n)).mean(-1, keepdims=True) + np.abs(g).mean(-1, keepdims=True)
        first = (eg + en * np.abs(g * n).mean(-1, keepdims=True)
                 + np.abs(n) * (np.abs(g) * en + np.abs(n) * eg).mean(-1, keepdims=True) + eg.mean(-1, keepdims=True))
        return r_ * (mag * K * U * 2 + first * 2)

    n, rx = T.normalised(_np(x), kind, EPS)
    en = _norm_error(_np(x), kind)
    w = np.abs(q.get("pre_weight", 1.0)) * np.ones_like(n)
    ee = back(gy * w, np.abs(gy) * w * U * 2, n, en, rx) + np.abs(want["x"]) * 2 * U
    _near(r.x, want["x"], ee, "grad x")
    rows = x.numel() // x.shape[-1]

    def sums(terms, errors):
        return (np.abs(terms) * (rows + K) * U + errors)

    if "pre_weight" in q:
        _near(r.pre_weight, want["pre_weight"], sums(gy * n, np.abs(gy) * en).sum(lead), "pre_weight")
    if "pre_bias" in q:
        _near(r.pre_bias, want["pre_bias"], sums(gy, 0 * gy).sum(lead), "pre_bias")
    e = want["x"]
    m, rb = T.normalised(_np(b), kind, EPS) if kw["post_norm"] else (_np(b), 1.0)
    em = _norm_error(_np(b), kind) if kw["post_norm"] else np.zeros_like(m)
    pw = np.abs(q.get("post_weight", 1.0)) * np.ones_like(m)
    s = np.abs(q.get("residual_scale", 1.0)) * np.ones_like(m)
    raw = q.get("gate", 1.0)
    a = np.abs(T.gate_act(raw, akw["gate_activation"])) * np.ones_like(m) if "gate" in q else np.ones_like(m)
    f = np.abs(m) * pw + np.abs(q.get("post_bias", 0.0))
    ef = em * pw + f * 4 * U
    h, eh = e * s * a, (ee + np.abs(e) * 8 * U) * s * a
    eb = back(h * pw, eh * pw, m, em, rb) if kw["post_norm"] else eh
    _near(r.branch, want["branch"], eb, "grad branch")
    if "post_weight" in q:
        _near(r.post_weight, want["post_weight"], sums(h * m, eh * np.abs(m) + np.abs(h) * em).sum(lead), "post_weight")
    if "post_bias" in q:
        _near(r.post_bias, want["post_bias"], sums(h, eh).sum(lead), "post_bias")
    if isinstance(p.get("residual_scale"), torch.Tensor):
        t = sums(e * a * f, (ee * f + np.abs(e) * ef) * a + np.abs(e) * a * f * 8 * U)
        _near(r.residual_scale, want["residual_scale"], T._sum_to(t, q["residual_scale"].shape) * (1 if p["residual_scale"].numel() > 1 else 2), "scale")
    elif "residual_scale" not in p or not isinstance(p["residual_scale"], torch.Tensor):
        assert r.residual_scale is None
    if "gate" in q:
        slope = np.abs(T.gate_slope(raw, akw["gate_activation"]))
        t = sums(e * s * f, (ee * f + np.abs(e) * ef) * s + np.abs(e) * s * f * (8 + K) * U)
        # The slope a (1 - a), 1 - a^2 from the float32 value: off by a few units of 1.
        _near(r.gate, want["gate"], T._sum_to(t, raw.shape) * slope + T._sum_to(np.abs(e * s * f), raw.shape) * 16 * U, "gate")
    for name in ("pre_weight", "pre_bias", "post_weight", "post_bias", "gate"):
        g = getattr(r, name)
        assert (g is None) == (name not in p)
        if g is not None:
            assert g.shape == p[name].shape and g.dtype == p[name].dtype
    again = rf.block_norm_backward(dx, dy, xs, bs, **kw, **akw, **p)
    for u, v in zip(r, again):
        assert u is None or torch.equal(u, v)
    return r


SHAPES = [(1, 1, 1), (1, 1, 768), (2, 3, 33), (3, 7, 256), (2, 5, 1000), (1, 4, 1024), (2, 3, 1025), (1, 2, 2304),
          (1, 3, 4096), (2, 2, 8200), (1, 2, 16384), (3, 40, 130), (2, 300, 64), (2, 100, 1100)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dt", list(TORCH))
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("post_norm", [True, False])
def test_shapes(shape, dt, kind, post_norm):
    x, b, p, kw, akw = _setup(shape, dt, kind, post_norm, "channel", None, "vector")
    _check_forward(x, b, p, kw, akw)
    _check_backward(x, b, p, kw, akw, _make(shape, dt, 10, 0.3), _make(shape, dt, 11, 0.3))


GATES = ["none", "channel", "sequence", "sequence_scalar", "token", "full", "one"]


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("act", [None, "sigmoid", "tanh"])
@pytest.mark.parametrize("scale", ["none", "number", "vector", "one"])
@pytest.mark.parametrize("shape", [(3, 40, 130), (2, 9, 1040), (20, 3, 72)], ids=str)
def test_gates_and_scales(gate, act, scale, shape):
    for kind, post_norm, pdt in (("rms", True, "float32"), ("layer", True, "bfloat16"), ("rms", False, "float16")):
        x, b, p, kw, akw = _setup(shape, "float32", kind, post_norm, gate, act, scale, pdt=pdt)
        _check_forward(x, b, p, kw, akw)
        _check_backward(x, b, p, kw, akw, _make(shape, "float32", 10, 0.3), _make(shape, "float32", 11, 0.3))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", list(TORCH))
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 3, 33), (2, 5, 1000), (1, 3, 4096), (3, 40, 130), (1, 2, 16384)], ids=str)
def test_saved(fmt, dt, shape):
    x, b, p, kw, akw = _setup(shape, dt, "rms", True, "channel", "sigmoid", "vector")
    _check_forward(x, b, p, kw, akw, save=fmt)
    _check_backward(x, b, p, kw, akw, _make(shape, dt, 10, 0.3), _make(shape, dt, 11, 0.3), save=fmt)


def test_one_sided_calls():
    import rollfast_b200 as rf

    shape = (2, 9, 200)
    x, b, p, kw, akw = _setup(shape, "float32", "layer", True, "channel", None, "vector")
    dx, dy = _make(shape, "float32", 10), _make(shape, "float32", 11)
    _check_backward(x, b, p, kw, akw, None, dy)
    _check_backward(x, b, p, kw, akw, dx, None)
    pre = {k: v for k, v in p.items() if k.startswith("pre")}
    r = rf.block_norm_forward(x, **kw, **pre)
    assert r.x is x
    want = T.block_norm(_np(x), None, _plain(pre), **kw)[1]
    _near(r.y, want, (_norm_error(_np(x), "layer") * np.abs(_np(pre["pre_weight"]))
                      + np.abs(_np(pre["pre_bias"])) * 4 * U + np.abs(want) * 4 * U), "y")
    g = rf.block_norm_backward(dx, dy, x, **kw, **pre)
    full = T.block_norm_grads(_np(dx), _np(dy), _np(x), None, _plain(pre), **kw)
    assert g.branch is None and g.gate is None
    for name in ("x", "pre_weight", "pre_bias"):
        assert np.allclose(_np(getattr(g, name)), full[name], rtol=1e-5, atol=1e-5)
    last = rf.block_norm_forward(x, b, pre_norm=False, **kw, **akw, **{k: v for k, v in p.items() if not k.startswith("pre")})
    assert last.y is None
    assert torch.equal(last.x, rf.block_norm_forward(x, b, **kw, **akw, **p).x)


def test_mixed_types_strides_and_no_rows():
    import rollfast_b200 as rf

    wide = _make((6, 5, 3 * 136), "bfloat16", 20)
    x = _make((6, 5, 136), "float32", 21)
    p = {"pre_weight": _make((136,), "bfloat16", 22, 0.1, 1.0), "post_weight": _make((136,), "float16", 23, 0.1, 1.0)}
    kw, akw = dict(kind="rms", eps=EPS, post_norm=True), {"gate_activation": None}
    for b in (wide[..., :136], wide[..., 136:272], wide[..., 1:137], wide[..., ::3], wide[:1, :, :136].expand(6, 5, 136)):
        r = _check_forward(x, b, p, kw, akw)
        assert r.x.dtype == torch.float32 and r.y.dtype == torch.bfloat16
        g = _check_backward(x, b, p, kw, akw, _make((6, 5, 136), "float32", 24), wide[..., 136:272])
        assert g.x.dtype == torch.float32 and g.branch.dtype == torch.bfloat16
    e = torch.empty(0, 136, device="cuda")
    r = rf.block_norm_forward(e, e.bfloat16(), **p, save="int8")
    assert r.x.shape == (0, 136) and r.y.shape == (0, 136) and r.saved_y.rows == 0
    gate = _make((136,), "float32", 25)
    g = rf.block_norm_backward(e, e, e, e, **p, gate=gate)
    assert (g.pre_weight == 0).all() and (g.post_weight == 0).all() and (g.gate == 0).all() and g.gate.shape == (136,)


def test_rows_that_are_zero_large_or_not_finite():
    """A row of zeros normalises to zeros; a large mean costs LayerNorm no
    digits of the deviations; a NaN stays in its row."""
    import rollfast_b200 as rf

    x = _make((8, 512), "float32", 30)
    x[1] = 0.0
    x[2] += 1000.0
    x[3, 7] = float("nan")
    for kind in ("rms", "layer"):
        y = rf.block_norm_forward(x, kind=kind, eps=1e-6).y
        assert (y[1] == 0).all() and y[3].isnan().all() and y[[0, 1, 2, 4, 5, 6, 7]].isfinite().all()
        n = T.normalised(_np(x), kind, 1e-6)[0]
        # float32 holds 1000 + z to 2^-14.1 of z's unit: the input is what is compared, so K U of the values taken.
        assert (np.abs(_np(y[2]) - n[2]) <= (np.abs(n[2]) + np.abs(_np(x[2])) * 2) * K * U).all()
        g = rf.block_norm_backward(torch.ones_like(x), torch.ones_like(x), x, kind=kind, eps=1e-6)
        assert g.x[3].isnan().all() and g.x[[0, 1, 2, 4, 5, 6, 7]].isfinite().all()


def test_captured_backward_follows_its_inputs():
    import rollfast_b200 as rf

    shape = (4, 50, 256)
    x, b, p, kw, akw = _setup(shape, "bfloat16", "rms", True, "sequence", "sigmoid", "vector")
    dx, dy = _make(shape, "bfloat16", 10), _make(shape, "bfloat16", 11)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        rf.block_norm_backward(dx, dy, x, b, **kw, **akw, **p)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        r = rf.block_norm_backward(dx, dy, x, b, **kw, **akw, **p)
    dx.mul_(2)
    dy.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    want = rf.block_norm_backward(dx, dy, x, b, **kw, **akw, **p)
    for u, v in zip(r, want):
        assert u is None or torch.equal(u, v)


@pytest.mark.parametrize("dt", list(TORCH))
def test_rms_with_biases(dt):
    shape = (2, 9, 264)
    x, b, p, kw, akw = _setup(shape, dt, "rms", True, "sequence", "tanh", "vector")
    p["pre_bias"], p["post_bias"] = _make((264,), "float32", 40, 0.2), _make((264,), "float32", 41, 0.2)
    _check_forward(x, b, p, kw, akw, save="e4m3")
    _check_backward(x, b, p, kw, akw, _make(shape, dt, 10, 0.3), _make(shape, dt, 11, 0.3))


def test_saved_and_unsaved_inputs_mix():
    """Either input saved, in either format, gives what its values give."""
    import rollfast_b200 as rf

    shape = (2, 30, 520)
    x, b, p, kw, akw = _setup(shape, "float32", "layer", True, "channel", None, "vector")
    dx, dy = _make(shape, "float32", 10), _make(shape, "float32", 11)
    sx, sb = rf.save_activation(x, "int8"), rf.save_activation(b, "e4m3")
    vx, vb = rf.load_activation(sx), rf.load_activation(sb)
    want = rf.block_norm_backward(dx, dy, vx, vb, **kw, **akw, **p)
    for pair in ((sx, sb), (sx, vb), (vx, sb)):
        got = rf.block_norm_backward(dx, dy, *pair, **kw, **akw, **p)
        for u, v in zip(got, want):
            assert torch.allclose(u, v, rtol=1e-4, atol=1e-5)
    only = rf.block_norm_backward(dx, None, sx, sb, **kw, **akw, **p)
    assert torch.equal(only.x, dx) and (only.pre_weight == 0).all()


def test_many_short_sequences():
    """More gate groups than the GPU holds at once, of two rows each."""
    shape = (3000, 2, 72)
    x, b, p, kw, akw = _setup(shape, "float32", "rms", True, "sequence", None, "one")
    _check_forward(x, b, p, kw, akw)
    _check_backward(x, b, p, kw, akw, _make(shape, "float32", 10, 0.3), _make(shape, "float32", 11, 0.3))


def test_rows_past_32_bit_offsets():
    import rollfast_b200 as rf

    rows, d = 300_001, 7_168  # 2.15e9 elements
    x = torch.zeros(rows, d, dtype=torch.bfloat16, device="cuda")
    x[-1] = _make((d,), "bfloat16", 50, 2.0)
    y = rf.block_norm_forward(x, eps=1e-6).y
    assert torch.equal(y[-1], rf.block_norm_forward(x[-1:].clone(), eps=1e-6).y[0])
    assert int((y[:-1] != 0).sum()) == 0
    g = torch.zeros_like(x)
    g[-1] = 1.0
    r = rf.block_norm_backward(None, g, x, eps=1e-6, pre_weight=torch.ones(d, device="cuda"))
    one = rf.block_norm_backward(None, g[-1:].clone(), x[-1:].clone(), eps=1e-6, pre_weight=torch.ones(d, device="cuda"))
    assert torch.equal(r.x[-1], one.x[0]) and torch.allclose(r.pre_weight, one.pre_weight, rtol=1e-6)
