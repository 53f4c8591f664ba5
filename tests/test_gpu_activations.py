"""Activations saved in 8 bits, the weight gradient and the SwiGLU that read
them, against the 64-bit plain forms (oracle/training_np.py).

Codes and steps are compared bit for bit.  Tolerances of computed results, by
arithmetic: a rounding to the output type is off by at most half a step,
finfo.eps / 2 relative to the value; the float32 work before it by a bound
stated at each test."""

import numpy as np
import pytest
import torch

from oracle import training_np as T

pytestmark = pytest.mark.gpu

TORCH = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
U = 2.0 ** -24  # half a unit of float32, relative


def _np(t):
    return t.detach().to(torch.float64).cpu().numpy()


def _half(dt):
    return torch.finfo(dt).eps / 2


def _tiny(dt):
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps


def _make(shape, dt, seed, scale=1.0):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal(shape) * np.exp(rng.standard_normal(shape[-1])) * scale
    return torch.from_numpy(x.astype(np.float32)).cuda().to(TORCH[dt])


def _codes_equal(saved, x, seed=None):
    rows, d = saved.rows, saved.features
    codes, scales = T.encode8(x.detach().float().cpu().numpy().reshape(rows, d), saved.format, seed)
    assert np.array_equal(saved.codes.cpu().numpy(), codes)
    assert np.array_equal(saved.scales.cpu().numpy()[:, :rows], scales[:, :rows])
    return T.decode8(codes, scales, d, saved.format).reshape(saved.shape)


SHAPES = [(1, 1), (5, 768), (3, 33), (65, 130), (2, 3, 1000), (1, 14336), (129, 17), (0, 40), (7, 2049), (40,)]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", list(TORCH))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("seed", [None, 0, 2 ** 64 - 3])
def test_save_and_load(fmt, dt, shape, seed):
    import rollfast_b200 as rf

    x = _make(shape, dt, 1)
    saved = rf.save_activation(x, fmt, seed=seed)
    assert saved.shape == shape and saved.dtype == x.dtype and saved.rows * saved.features == x.numel()
    v = _codes_equal(saved, x, seed)
    for out_dt in TORCH.values():
        got = rf.load_activation(saved, dtype=out_dt)
        assert got.shape == x.shape and got.dtype == out_dt
        most = torch.finfo(out_dt).max
        want = torch.from_numpy(np.clip(v, -most, most)).to(torch.float32).to(out_dt)
        assert torch.equal(got.cpu(), want)
    assert rf.load_activation(saved).dtype == x.dtype


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("seed", [None, 99])
def test_special_values(fmt, seed):
    import rollfast_b200 as rf

    x = torch.zeros(12, 96)
    x[1, 3], x[2, 40], x[3, 95] = float("inf"), float("nan"), -float("inf")
    x[4] = 3.4e38
    x[5] = torch.finfo(torch.float32).max
    x[6, :5] = 1e-40
    x[7] = 2.0 ** -126
    x[8] = 127.0
    x[9] = 448.0
    x[10, 0] = 127.0001
    x[11] = -0.0
    x = x.cuda()
    saved = rf.save_activation(x, fmt, seed=seed)
    v = _codes_equal(saved, x, seed)
    got = rf.load_activation(saved).cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(v))
    fine = ~np.isnan(v)
    assert np.array_equal(got[fine], v[fine].astype(np.float32))
    assert np.isfinite(got[4:]).all()
    half = rf.load_activation(saved, dtype=torch.float16)
    assert (half[4] == 65504).all() and half[1].isnan().sum() == 32


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["bfloat16", "float32"])
@pytest.mark.parametrize("features", [256, 250])
@pytest.mark.parametrize("seed", [None, 7])
def test_wide_and_tiny_ranges_within_a_block(fmt, dt, features, seed):
    """Magnitudes from the type's least to the block's largest, at largest
    values of 2^-130 to 2^-1: below a step, subnormal in the code, and zeros."""
    import rollfast_b200 as rf

    rng = np.random.default_rng(11)
    top = -130 + np.arange(130)[:, None]
    low = np.maximum(top - 18, -133)
    e = low + np.floor(rng.random((130, features)) * (top - low + 1))
    v = np.ldexp(rng.choice([-1.0, 1.0], e.shape), e.astype(int)) * (rng.random(e.shape) > 0.1)
    x = torch.from_numpy(v).to(torch.float32).cuda().to(TORCH[dt])
    _codes_equal(rf.save_activation(x, fmt, seed=seed), x, seed)


def test_row_strided_views_are_read_in_place():
    import rollfast_b200 as rf

    both = _make((37, 2 * 200), "bfloat16", 2)
    for x in (both[:, :200], both[:, 200:], both[::3, 8:72], both[:, 1:34], both.t()[:50], both[:1].expand(9, 400)):
        _codes_equal(rf.save_activation(x), x)


def test_saved_rows_past_32_bit_offsets():
    import rollfast_b200 as rf

    rows, d = 150_001, 14_400  # 2.16e9 codes
    x = torch.zeros(rows, d, dtype=torch.bfloat16, device="cuda")
    x[-1] = _make((d,), "bfloat16", 3)
    x[rows // 2, 7] = 3.0
    saved = rf.save_activation(x)
    codes, scales = T.encode8(x[-1:].float().cpu().numpy(), "int8")
    assert np.array_equal(saved.codes[-1:].cpu().numpy(), codes)
    assert np.array_equal(saved.scales[:, rows - 1].cpu().numpy(), scales[:, 0])
    del x
    back = rf.load_activation(saved)
    assert back[rows // 2, 7] == 3.0 and int((back[: rows - 1] != 0).sum()) == 1
    assert np.array_equal(_np(back[-1]), T.decode8(codes, scales, d, "int8")[0])
    del back
    g = torch.zeros(rows, 8, dtype=torch.bfloat16, device="cuda")
    g[-1] = 1.0
    got = _np(rf.weight_gradient(saved, g))
    assert np.array_equal(got, np.repeat(T.decode8(codes, scales, d, "int8").T, 8, axis=1))


WGRAD = [  # rows, in, out
    (1, 1, 1), (1, 40, 24), (64, 128, 256), (65, 129, 257), (333, 768, 768), (63, 300, 16), (500, 16, 700),
    (1025, 260, 250), (4100, 513, 77), (7, 1000, 1391), (20000, 96, 64),
]


def _wgrad_bound(x, g, terms, dt, want):
    # A sum of T float32 additions, each off by at most one unit (2 U: the
    # tensor cores may truncate), of exact products; partial sums of a split
    # and the terms of G add as many again.  Then the output's rounding.
    s = np.abs(x).reshape(-1, x.shape[-1]).T @ np.abs(g).reshape(-1, g.shape[-1])
    n = x.reshape(-1, x.shape[-1]).shape[0] * terms + 70
    return n * 2 * U * s + np.abs(want) * _half(dt) + _tiny(dt)


@pytest.mark.parametrize("shape", WGRAD, ids=str)
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", list(TORCH))
@pytest.mark.parametrize("layout", ["io", "oi"])
@pytest.mark.parametrize("out_dt,initial", [("float32", False), ("float32", True), ("bfloat16", True)])
def test_weight_gradient(shape, fmt, dt, layout, out_dt, initial):
    import rollfast_b200 as rf

    rows, k, n = shape
    saved = rf.save_activation(_make((rows, k), dt, 4), fmt)
    x = T.decode8(saved.codes.cpu().numpy(), saved.scales.cpu().numpy(), k, fmt)
    g = _make((rows, n), dt, 5, 0.1)
    out_shape = (k, n) if layout == "io" else (n, k)
    init = _make(out_shape, out_dt, 6) if initial else None
    got = rf.weight_gradient(saved, g, initial=init, layout=layout, dtype=TORCH[out_dt])
    assert got.shape == out_shape and got.dtype == TORCH[out_dt]
    want = T.weight_gradient(x, _np(g), None if init is None else _np(init), layout)
    bound = _wgrad_bound(x, _np(g), {"bfloat16": 1, "float16": 2, "float32": 3}[dt], got.dtype,
                         want if layout == "io" else want.T)
    bound = bound if layout == "io" else bound.T
    if init is not None:
        bound = bound + np.abs(_np(init)) * 2 * U
    assert (np.abs(_np(got) - want) <= bound).all()
    # The same operands give the same bits, and in-place accumulation the same sum.
    again = rf.weight_gradient(saved, g, initial=init, layout=layout, dtype=TORCH[out_dt])
    assert torch.equal(got, again)
    if init is not None:
        same = rf.weight_gradient(saved, g, initial=init, out=init, layout=layout)
        assert same is init and torch.equal(init, got)


def test_weight_gradient_is_exact_on_whole_numbers():
    """Small integers: every product and partial sum is exact in float32, so
    the result must be equal, whatever the order of the sum."""
    import rollfast_b200 as rf

    rng = np.random.default_rng(7)
    for rows, k, n in [(1000, 640, 520), (129, 31, 1030)]:
        x = torch.from_numpy(rng.integers(-100, 101, (rows, k)).astype(np.float32)).cuda()
        x[:, 0] = 127.0  # every first block's step is 1
        g = torch.from_numpy(rng.integers(-8, 9, (rows, n)).astype(np.float32)).cuda()
        saved = rf.save_activation(x)
        xs = T.decode8(saved.codes.cpu().numpy(), saved.scales.cpu().numpy(), k, "int8")
        for dt in TORCH.values():
            for layout in ("io", "oi"):
                got = rf.weight_gradient(saved, g.to(dt), layout=layout)
                assert np.array_equal(_np(got), T.weight_gradient(xs, _np(g), layout=layout))


def test_weight_gradient_without_rows():
    import rollfast_b200 as rf

    saved = rf.save_activation(torch.zeros(0, 40, dtype=torch.bfloat16, device="cuda"))
    g = torch.zeros(0, 24, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(rf.weight_gradient(saved, g), torch.zeros(40, 24, device="cuda"))
    init = _make((40, 24), "float32", 8)
    assert torch.equal(rf.weight_gradient(saved, g, initial=init), init)


def test_weight_gradient_poison_and_infinities():
    """A NaN block reaches its 32 rows of the result only; an infinite
    gradient its column; tokens behind the last reach nothing."""
    import rollfast_b200 as rf

    x = _make((70, 256), "bfloat16", 9)
    g = _make((70, 130), "bfloat16", 10)
    x[69, 40] = float("nan")
    saved = rf.save_activation(x)
    saved.scales[:, 70:] = 255  # steps of rows that do not exist
    got = rf.weight_gradient(saved, g)
    assert got[32:64].isnan().all() and got[:32].isfinite().all() and got[64:].isfinite().all()
    for dt in TORCH.values():
        h = g.to(dt)
        h[3, 5] = float("inf")
        clean = rf.save_activation(_make((70, 256), "bfloat16", 11).abs() + 1)
        got = rf.weight_gradient(clean, h)
        assert (got[:, 5] == float("inf")).all()
        assert got[:, :5].isfinite().all() and got[:, 6:].isfinite().all()


def test_weight_gradient_strides_and_outputs():
    import rollfast_b200 as rf

    x = _make((4, 25, 96), "bfloat16", 12)
    wide = _make((4, 25, 3 * 72), "bfloat16", 13)
    saved = rf.save_activation(x)
    xs = _np(rf.load_activation(saved))
    buf = torch.full((100, 200), 7.0, device="cuda")
    for g in (wide[..., :72], wide[..., 72:144], wide[..., 1:73], wide[:, :, ::3], wide[:1, :, :72].expand(4, 25, 72)):
        out = buf[2:98, 3:75]
        got = rf.weight_gradient(saved, g, out=out)
        assert got is out
        want = T.weight_gradient(xs, _np(g))
        assert (np.abs(_np(out) - want) <= _wgrad_bound(xs, _np(g), 1, torch.float32, want)).all()
        assert (buf[:2] == 7).all() and (buf[98:] == 7).all() and (buf[:, :3] == 7).all() and (buf[:, 75:] == 7).all()
    init = _make((96, 72), "float32", 14)
    got = rf.weight_gradient(saved, wide[..., :72], initial=init, out=buf[2:98, 3:75])
    want = T.weight_gradient(xs, _np(wide[..., :72]), _np(init))
    assert np.allclose(_np(got), want, rtol=0, atol=1e-3)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", list(TORCH))
@pytest.mark.parametrize("shape", [(1, 1), (5, 768), (3, 33), (65, 130), (2, 3, 1000), (0, 40)], ids=str)
def test_swiglu(fmt, dt, shape):
    import rollfast_b200 as rf

    both = _make((*shape[:-1], 2 * shape[-1]), dt, 15, 2.0)
    gate, up = both[..., :shape[-1]], both[..., shape[-1]:]
    h, sg, su = rf.swiglu_forward(gate, up, fmt)
    vg, vu = _codes_equal(sg, gate), _codes_equal(su, up)
    g, u = _np(gate), _np(up)
    want = T.swiglu(g, u)
    # exp(-g) is off by at most 2 + 1.2 |g| units of float32, the sigmoid by as
    # much and a few roundings, the products by two more.
    rel = (8 + 2 * np.abs(g)) * 2 * U
    with np.errstate(over="ignore"):
        most = torch.finfo(TORCH[dt]).max
    ok = np.abs(want) < most
    assert (np.abs(_np(h) - want) <= np.abs(want) * (rel + _half(TORCH[dt])) + 2 * _tiny(TORCH[dt]))[ok].all()
    assert rf.swiglu_forward(gate, up, None)[1:] == (None, None)
    assert torch.equal(rf.swiglu_forward(gate, up, None)[0], h)

    d = _make(shape, dt, 16, 0.1)
    dg, du, sh = rf.swiglu_backward(d, sg, su, save_h=fmt)
    wg, wu = T.swiglu_grads(_np(d), vg, vu)
    dn = np.abs(_np(d))
    # The slope s + a (1 - s) cancels where it is near 0: its error is that of its summands.
    err = (1 + np.abs(vg)) * (8 + 2 * np.abs(vg)) * 4 * U
    half, tiny = _half(TORCH[dt]), 2 * _tiny(TORCH[dt])
    assert (np.abs(_np(dg) - wg) <= dn * np.abs(vu) * err + np.abs(wg) * half + tiny).all()
    assert (np.abs(_np(du) - wu) <= dn * np.abs(vg) * err + np.abs(wu) * half + tiny).all()
    # h again: within the code's own half step of the float32 product.
    wh = T.swiglu(vg, vu)
    got = T.decode8(sh.codes.cpu().numpy(), sh.scales.cpu().numpy(), sh.features, fmt).reshape(shape)
    s = sh.scales.cpu().numpy()[:, :sh.rows].transpose(1, 0, 2).reshape(sh.rows, sh.scales.shape[0] * 4).astype(int)
    step = np.repeat(2.0 ** (s - 127.0), 32, axis=1)[:, :sh.features].reshape(shape)
    grid = step / 2 if fmt == "int8" else np.maximum(np.abs(wh) * 2.0 ** -4, step * 2.0 ** -10)
    assert (np.abs(got - wh) <= grid + np.abs(wh) * (8 + 2 * np.abs(vg)) * 2 * U).all()
    # Into the halves of a fused gradient.
    fused = torch.full((*shape[:-1], 2 * shape[-1] + 3), 5.0, dtype=TORCH[dt], device="cuda")
    out = rf.swiglu_backward(d, sg, su, grad_gate=fused[..., :shape[-1]], grad_up=fused[..., shape[-1]:2 * shape[-1]])
    assert torch.equal(out[0], dg) and torch.equal(out[1], du) and out[2] is None
    assert (fused[..., 2 * shape[-1]:] == 5).all()


def test_swiglu_far_inputs():
    import rollfast_b200 as rf

    g = torch.tensor([[-200.0, -90.0, -20.0, 0.0, 20.0, 90.0, 200.0, 1e30]], device="cuda")
    u = torch.ones_like(g)
    h, sg, su = rf.swiglu_forward(g, u)
    assert h.isfinite().all() and (h[0, 4:] == g[0, 4:]).all() and (h[0, :2].abs() < 1e-30).all()
    dg, du, _ = rf.swiglu_backward(torch.ones_like(g), sg, su)
    assert dg.isfinite().all() and du.isfinite().all()


def test_another_stream_and_graph_replay():
    """The calls run on the current stream; captured calls follow changed
    inputs at replay, two graphs do not share workspaces."""
    import rollfast_b200 as rf

    x = _make((700, 192), "float32", 17)
    g = _make((700, 96), "float32", 18)
    want = rf.weight_gradient(rf.save_activation(x), g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = rf.weight_gradient(rf.save_activation(x), g)
    s.synchronize()
    assert torch.equal(got, want)

    graphs, outs, ins = [], [], []
    for i in range(2):
        a, b = x.clone(), g.clone()
        with torch.cuda.stream(s):
            rf.weight_gradient(rf.save_activation(a), b)  # warm
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(rf.weight_gradient(rf.save_activation(a), b))
        graphs.append(graph)
        ins.append((a, b))
    ins[0][0].mul_(2.0)
    ins[1][1].mul_(-4.0)
    torch.cuda.synchronize()
    t = torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(s):
            graphs[0].replay()
        with torch.cuda.stream(t):
            graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want * 2) and torch.equal(outs[1], want * -4)


def test_no_device_side_wait_gave_up():
    from rollfast_b200 import _lib

    torch.cuda.synchronize()
    _lib.sync_check(torch.cuda.current_stream().cuda_stream)


def test_swiglu_of_two_formats_and_shared_gradients():
    import rollfast_b200 as rf

    g, u, d = (_make((33, 264), "bfloat16", s) for s in (20, 21, 22))
    sg, su = rf.save_activation(g, "int8"), rf.save_activation(u, "e4m3")
    dg, du, sh = rf.swiglu_backward(d, sg, su, save_h="int8")
    vg, vu = rf.load_activation(sg), rf.load_activation(su)
    wg, wu = T.swiglu_grads(_np(d), _np(vg), _np(vu))
    assert np.allclose(_np(dg), wg, rtol=2.0 ** -7, atol=1e-5) and np.allclose(_np(du), wu, rtol=2.0 ** -7, atol=1e-5)
    with pytest.raises(ValueError):
        rf.swiglu_backward(d, sg, su, grad_gate=dg, grad_up=dg)
    # In place over the incoming gradient.
    e = d.clone()
    got = rf.swiglu_backward(e, sg, su, grad_gate=e)
    assert got[0] is e and torch.equal(e, dg) and torch.equal(got[1], du)


def test_weight_gradient_of_many_shapes_on_whole_numbers():
    """Tiles whole and in parts, one and several waves of them, odd edges."""
    import rollfast_b200 as rf

    rng = np.random.default_rng(23)
    for rows, k, n in [(2050, 768, 300), (129, 2600, 2050), (4097, 30, 5000), (300, 5000, 2304), (10000, 257, 257)]:
        x = torch.from_numpy(rng.integers(-3, 4, (rows, k)).astype(np.float32)).cuda()
        x[:, ::32] = 127.0
        g = torch.from_numpy(rng.integers(-2, 3, (rows, n)).astype(np.float32)).cuda().bfloat16()
        saved = rf.save_activation(x.bfloat16())
        want = (rf.load_activation(saved, dtype=torch.float32).double().t() @ g.double()).float()
        assert torch.equal(rf.weight_gradient(saved, g), want)
        assert torch.equal(rf.weight_gradient(saved, g, layout="oi"), want.t())
