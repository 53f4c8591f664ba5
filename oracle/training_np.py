"""64-bit plain forms of the training-step operators (8-bit activations,
weight gradient, SwiGLU, block norms) -- TEST INFRASTRUCTURE ONLY.

No reference counterpart.  The 8-bit form is restated from its definition
(``include/rollfast_b200.h``, ``rf_saved_activation``); the gradients are the
formulas, checked against differences by ``tests/test_training_oracle.py``.
"""

import numpy as np

from .muon_np import splitmix64

FORMATS = {"int8": (127.0, 248), "e4m3": (448.0, 246)}

# The magnitudes of the e4m3 codes 0 .. 126 (127 is a NaN).
_E4M3 = np.array([(m / 8 * 2.0 ** -6) if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127])


def noise16(seed, n):
    """n numbers in [0, 1) of 16 bits: output c of the seed's SplitMix64 sequence serves elements 4c .. 4c + 3."""
    with np.errstate(over="ignore"):
        c = np.arange((n + 3) // 4, dtype=np.uint64)
        z = splitmix64(np.uint64(seed) + c * np.uint64(0x9E3779B97F4A7C15))
    parts = np.stack([(z >> np.uint64(16 * j)) & np.uint64(0xFFFF) for j in range(4)], axis=1)
    return parts.reshape(-1)[:n].astype(np.float64) / 65536


def encode8(x, fmt, seed=None):
    """x (rows, features), float32 values -> (codes (rows, ld) uint8, scales (panels, rows up to 64, 4) uint8)."""
    x = np.asarray(x, np.float32)
    rows, features = x.shape
    most, top = FORMATS[fmt]
    panels, ld = -(-features // 128), -(-features // 16) * 16
    b = np.zeros((rows, panels * 128), np.float32)
    b[:, :features] = x
    b = b.reshape(rows, panels * 4, 32)
    fine = np.isfinite(b).all(-1)
    a = np.where(fine, np.abs(b).max(-1), 0).astype(np.float64)
    with np.errstate(divide="ignore"):
        m, e = np.frexp(a / most)  # a <= most * 2^k for k = e, or e - 1 where m is 1/2 exactly
    s = np.where(a > 0, e - (m == 0.5) + 127, 1).clip(1, top)
    v = np.where(fine[..., None], b, 0).astype(np.float64) * 2.0 ** (127 - s)[..., None]
    u = None
    if seed is not None:
        u = np.zeros((rows, panels * 128))
        u[:, :features] = noise16(seed, rows * features).reshape(rows, features)
        u = u.reshape(b.shape)
    if fmt == "int8":
        # The sum of value and noise is one float32 addition.
        q = np.rint(v) if u is None else np.floor((v.astype(np.float32) + u.astype(np.float32)).astype(np.float64))
        codes = q.clip(-127, 127).astype(np.int8).view(np.uint8)
    else:
        w = np.minimum(np.abs(v), most)
        with np.errstate(divide="ignore"):
            step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(w, 2.0 ** -20))), -6) - 3)
        g = w / step
        g = np.rint(g) if u is None else np.floor((g.astype(np.float32) + u.astype(np.float32)).astype(np.float64))
        codes = np.searchsorted(_E4M3, np.minimum(g * step, most)).astype(np.uint8)
        codes |= (np.signbit(v) & fine[..., None]).astype(np.uint8) << 7
    codes = codes.reshape(rows, panels * 128)[:, :ld].copy()
    scales = np.ones((panels, -(-rows // 64) * 64, 4), np.uint8)
    scales[:, :rows] = np.where(fine, s, 255).astype(np.uint8).reshape(rows, panels, 4).transpose(1, 0, 2)
    return codes, scales


def decode8(codes, scales, features, fmt):
    """The values, float64 (rows, features)."""
    rows = codes.shape[0]
    if fmt == "int8":
        v = codes.view(np.int8).astype(np.float64)
    else:
        v = _E4M3[codes & 127] * np.where(codes & 128, -1.0, 1.0)
    s = scales[:, :rows].transpose(1, 0, 2).reshape(rows, scales.shape[0] * 4).astype(np.int64)
    step = np.where(s == 255, np.nan, 2.0 ** (s - 127))
    return (v * np.repeat(step, 32, axis=1)[:, :codes.shape[1]])[:, :features]


def weight_gradient(x, g, initial=None, layout="io"):
    x, g = np.asarray(x, np.float64), np.asarray(g, np.float64)
    w = x.reshape(-1, x.shape[-1]).T @ g.reshape(-1, g.shape[-1])
    w = w if layout == "io" else w.T
    return w if initial is None else w + initial


def sigmoid(g):
    g = np.asarray(g, np.float64)
    e = np.exp(-np.abs(g))  # no overflow, and no cancellation where the result is small
    return np.where(g < 0, e, 1.0) / (1 + e)


def swiglu(g, u):
    return g * sigmoid(g) * u


def swiglu_grads(dh, g, u):
    s = sigmoid(g)
    return dh * u * s * (1 + g * (1 - s)), dh * g * s


def gate_act(g, name):
    return sigmoid(g) if name == "sigmoid" else np.tanh(g) if name == "tanh" else g


def gate_slope(g, name):
    a = gate_act(g, name)
    return a * (1 - a) if name == "sigmoid" else 1 - a * a if name == "tanh" else np.ones_like(g)


def normalised(v, kind, eps):
    v = np.asarray(v, np.float64)
    if kind == "layer":
        v = v - v.mean(-1, keepdims=True)
    r = 1 / np.sqrt((v * v).mean(-1, keepdims=True) + eps)
    return v * r, r


def _one(p, name, absent):
    return absent if p.get(name) is None else np.asarray(p[name], np.float64)


def block_norm(x, branch, p, kind="rms", eps=1e-6, post_norm=True, gate_activation=None):
    """(x', y); p holds the parameters by the product's argument names."""
    x = np.asarray(x, np.float64)
    if branch is not None:
        n = normalised(branch, kind, eps)[0] if post_norm else np.asarray(branch, np.float64)
        n = n * _one(p, "post_weight", 1.0) + _one(p, "post_bias", 0.0)
        if p.get("gate") is not None:
            n = n * gate_act(_one(p, "gate", 1.0), gate_activation)
        x = x + _one(p, "residual_scale", 1.0) * n
    return x, normalised(x, kind, eps)[0] * _one(p, "pre_weight", 1.0) + _one(p, "pre_bias", 0.0)


def _sum_to(v, shape):
    """Sums a broadcast array's gradient back to its shape."""
    shape = tuple(shape)
    v = v.sum(tuple(range(v.ndim - len(shape)))) if v.ndim > len(shape) else v
    over = tuple(i for i, n in enumerate(shape) if n == 1 and v.shape[i] != 1)
    return v.sum(over, keepdims=True) if over else v


def block_norm_grads(dx, dy, x, branch, p, kind="rms", eps=1e-6, post_norm=True, gate_activation=None):
    """Gradients by argument name; x is x'."""
    x = np.asarray(x, np.float64)
    dx = np.zeros_like(x) if dx is None else np.asarray(dx, np.float64)
    dy = np.zeros_like(x) if dy is None else np.asarray(dy, np.float64)
    lead = tuple(range(x.ndim - 1))

    def back(g, n, r):
        g = g - n * (g * n).mean(-1, keepdims=True) - (g.mean(-1, keepdims=True) if kind == "layer" else 0.0)
        return g * r

    out = {}
    n, r = normalised(x, kind, eps)
    out["pre_weight"], out["pre_bias"] = (dy * n).sum(lead), dy.sum(lead)
    e = dx + back(dy * _one(p, "pre_weight", 1.0), n, r)
    out["x"] = e
    if branch is None:
        return {k: v for k, v in out.items() if k == "x" or p.get(k) is not None}
    m, rb = normalised(branch, kind, eps) if post_norm else (np.asarray(branch, np.float64), None)
    w, s = _one(p, "post_weight", 1.0), _one(p, "residual_scale", 1.0)
    f = m * w + _one(p, "post_bias", 0.0)
    raw = _one(p, "gate", 1.0)
    a = gate_act(raw, gate_activation) if p.get("gate") is not None else np.float64(1.0)
    if p.get("gate") is not None:
        out["gate"] = _sum_to(e * s * f * np.ones_like(e), raw.shape) * gate_slope(raw, gate_activation)
    if p.get("residual_scale") is not None and np.ndim(p["residual_scale"]):
        out["residual_scale"] = _sum_to(e * a * f, np.shape(p["residual_scale"]))
    h = e * a * s
    out["post_weight"], out["post_bias"] = (h * m).sum(lead), (h * np.ones_like(x)).sum(lead)
    out["branch"] = back(h * w, m, rb) if post_norm else h
    return {k: v for k, v in out.items() if k in ("x", "branch") or p.get(k) is not None}
