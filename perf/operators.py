"""The operators of a block's training step around the optimizer, as they are timed and compared.

Four operators: activations kept in 8 bits between the forward and the backward pass (``save_activation``,
``load_activation``), the weight gradient read straight from them (``weight_gradient``), a SwiGLU that keeps its two
inputs in 8 bits (``swiglu_forward``, ``swiglu_backward``), and the norms after one block and before the next, joined by
the gate, the residual scale and the residual addition (``block_norm_forward``, ``block_norm_backward``).

8-bit form.  A row of features is cut into blocks of 32.  A block holds 32 codes (two's complement ``int8``, or
``e4m3``) and one byte s, the biased exponent of its power-of-two step: value = code * 2^(s - 127).  s is the smallest in
[1, top] with max|x| <= 127 * 2^(s - 127) (448 for e4m3; top 248 and 246, the largest at which every code is finite in
float32 and bfloat16); s = 255 marks a block with an infinity or a NaN, and all of it reads as NaN.  Codes are
(rows, features rounded up to 16) bytes; the bytes s are (panels of 128 features, rows rounded up to 64, 4).
"""

import torch

own = False

# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
# Widths are those of the repository's two model shapes (768 and 768 x 2304; 4096, 1024 and 4096 x 14336) and odd ones.


def listed():
    return [
        # One short sequence's last tokens in a small model: what counts is the time to launch.
        dict(name="save_load_5x768", op="save", rows=5, features=768, dtype="bfloat16", format="int8", stochastic=False),
        # A long micro-batch's feed-forward activation, rounded stochastically so that gradients stay unbiased.
        dict(name="save_load_16384x14336_sr", op="save", rows=16384, features=14336, dtype="bfloat16", format="e4m3",
             stochastic=True),
        # A projection of a small model over a short, odd number of tokens.
        dict(name="wgrad_333x768x768", op="wgrad", rows=333, features=768, out=768, dtype="bfloat16", format="int8",
             layout="io", out_dtype="float32", initial=False),
        # Ragged in every direction, float32 gradients added to an accumulated one, stored (out, in).
        dict(name="wgrad_1537x1000x1391_f32", op="wgrad", rows=1537, features=1000, out=1391, dtype="float32",
             format="int8", layout="oi", out_dtype="float32", initial=True),
        # Few output tiles over many tokens: the fused q, k, v projection of a small model.
        dict(name="wgrad_32768x768x2304", op="wgrad", rows=32768, features=768, out=2304, dtype="bfloat16",
             format="e4m3", layout="io", out_dtype="bfloat16", initial=False),
        # The gate or up projection of a large model, accumulated over micro-batches.
        dict(name="wgrad_8192x4096x14336", op="wgrad", rows=8192, features=4096, out=14336, dtype="bfloat16",
             format="int8", layout="io", out_dtype="float32", initial=True),
        # The feed-forward block of a large model, forward and backward.
        dict(name="swiglu_fwd_8192x14336", op="swiglu_fwd", rows=8192, features=14336, dtype="bfloat16", format="int8"),
        dict(name="swiglu_bwd_8192x14336", op="swiglu_bwd", rows=8192, features=14336, dtype="bfloat16", format="int8"),
        # Between two blocks of a small model, a few tokens: LayerNorm with biases before the next block only.
        dict(name="norm_fwd_4x768", op="norm_fwd", batch=1, seq=4, features=768, dtype="bfloat16", kind="layer",
             post_norm=False, affine=True, gate="none", gate_activation="none", scale="none", save="none"),
        # Between two blocks of a large model: both norms, a gate per channel, a learned scale, 8-bit copies kept.
        dict(name="norm_fwd_16384x4096_saved", op="norm_fwd", batch=4, seq=4096, features=4096, dtype="bfloat16",
             kind="rms", post_norm=True, affine=True, gate="channel", gate_activation="none", scale="vector",
             save="int8"),
        # Odd sizes in float32, LayerNorms with biases, a sigmoid gate for each sequence.
        dict(name="norm_bwd_3x509x1001_f32", op="norm_bwd", batch=3, seq=509, features=1001, dtype="float32",
             kind="layer", post_norm=True, affine=True, gate="sequence", gate_activation="sigmoid", scale="vector",
             save="none"),
        # The backward pass of the large one, reading the 8-bit copies.
        dict(name="norm_bwd_16384x4096_saved", op="norm_bwd", batch=4, seq=4096, features=4096, dtype="bfloat16",
             kind="rms", post_norm=True, affine=True, gate="channel", gate_activation="none", scale="vector",
             save="int8"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["save", "wgrad", "wgrad", "swiglu_fwd", "swiglu_bwd", "norm_fwd", "norm_bwd"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    fmt = rng.choice(["int8", "e4m3"])
    if op == "wgrad":
        rows = _log(rng, 1, 65536)
        features, out = _log(rng, 16, 14336), _log(rng, 16, 14336)
        most = 8192 * 4096 * 14336 // {"bfloat16": 1, "float16": 2, "float32": 3}[dtype]
        rows = max(1, min(rows, most // (features * out)))
        return dict(op=op, rows=rows, features=features, out=out, dtype=dtype, format=fmt,
                    layout=rng.choice(["io", "oi"]), out_dtype=rng.choice(["float32", "bfloat16"]),
                    initial=rng.choice([False, True]))
    if op in ("save", "swiglu_fwd", "swiglu_bwd"):
        features = _log(rng, 8, 28672)
        rows = min(_log(rng, 1, 65536), 8192 * 14336 // 2 // features)
        case = dict(op=op, rows=rows, features=features, dtype=dtype, format=fmt)
        if op == "save":
            case["stochastic"] = rng.choice([False, True])
        return case
    features = _log(rng, 32, 16384)
    rows = min(_log(rng, 1, 65536), 16384 * 4096 // 2 // features)
    batch = rng.choice([1, 2, 3, 8])
    post = rng.choice([True, True, False])
    return dict(op=op, batch=batch, seq=max(1, rows // batch), features=features, dtype=dtype,
                kind=rng.choice(["rms", "rms", "layer"]), post_norm=post, affine=rng.choice([True, True, False]),
                gate=rng.choice(["none", "channel", "sequence", "token", "full"]),
                gate_activation=rng.choice(["none", "sigmoid", "tanh"]),
                scale=rng.choice(["none", "number", "vector"]), save=rng.choice(["none", "none", "int8", "e4m3"]))


_DTYPE = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}


def work(case):
    op, e = case["op"], _SIZE[case["dtype"]]
    q = 1 + 1 / 32  # bytes of an element in 8 bits, with its share of the block's exponent
    if op == "wgrad":
        t, k, n, o = case["rows"], case["features"], case["out"], _SIZE[case["out_dtype"]]
        return {"bytes": t * k * q + t * n * e + k * n * o * (2 if case["initial"] else 1), "flops": 2 * t * k * n}
    if op == "save":
        n = case["rows"] * case["features"]
        return {"bytes": n * (2 * e + 2 * q), "flops": n * 4}
    if op == "swiglu_fwd":
        # gate and up read, h and both 8-bit copies written, and the copies read back as values.
        n = case["rows"] * case["features"]
        return {"bytes": n * (3 * e + 2 * q + 2 * (q + e)), "flops": n * 12}
    if op == "swiglu_bwd":
        # dh and both copies read, both gradients and h's copy written, and that read back as values.
        n = case["rows"] * case["features"]
        return {"bytes": n * (3 * e + 3 * q + q + e), "flops": n * 20}
    n = case["batch"] * case["seq"] * case["features"]
    gate = n * e if case["gate"] == "full" else 0
    kept = 0 if case["save"] == "none" else 1
    if op == "norm_fwd":
        return {"bytes": n * 4 * e + gate + kept * n * 3 * (2 * q + e), "flops": n * 16}
    return {"bytes": n * (4 * e + 2 * (q if kept else e)) + 2 * gate, "flops": n * 30}


# ---------------------------------------------------------------------------
# The 8-bit form with elementary operations
# ---------------------------------------------------------------------------
_BITS = {"int8": (6, 0x7E0000, 248), "e4m3": (8, 0x600000, 246)}


def _noise(n, seed, device):
    """16 bits for each of n elements: output c of the SplitMix64 sequence of the seed serves elements 4c .. 4c+3."""
    def signed(v):
        v &= (1 << 64) - 1
        return v - (1 << 64) if v >= 1 << 63 else v

    def shifted(z, k):
        return (z >> k) & ((1 << (64 - k)) - 1)

    c = torch.arange((n + 3) // 4, device=device, dtype=torch.int64)
    z = (c + 1) * signed(0x9E3779B97F4A7C15) + signed(seed)
    z = (z ^ shifted(z, 30)) * signed(0xBF58476D1CE4E5B9)
    z = (z ^ shifted(z, 27)) * signed(0x94D049BB133111EB)
    z = z ^ shifted(z, 31)
    parts = torch.stack([shifted(z, 16 * j) & 0xFFFF if j else z & 0xFFFF for j in (0, 1, 2, 3)], dim=1)
    return parts.reshape(-1)[:n].to(torch.float32) / 65536


def _quantise(x, fmt, seed=None):
    """x (rows, features) in float32 -> (codes as numbers (rows, blocks, 32), exponents s (rows, blocks))."""
    rows, features = x.shape
    shift, border, top = _BITS[fmt]
    pad = -features % 32
    b = torch.nn.functional.pad(x, (0, pad)).reshape(rows, -1, 32)
    a = b.abs().amax(-1)
    fine = torch.isfinite(b).all(-1)
    bits = torch.where(fine, a, torch.zeros_like(a)).view(torch.int32)
    s = ((bits >> 23) - shift + ((bits & 0x7FFFFF) > border).to(torch.int32)).clamp(1, top)
    v = torch.where(fine[..., None], b, torch.zeros_like(b)) * ((254 - s) << 23).view(torch.float32)[..., None]
    if seed is not None:
        u = torch.nn.functional.pad(_noise(rows * features, seed, x.device).reshape(rows, features), (0, pad))
        u = u.reshape(b.shape)
    if fmt == "int8":
        v = (torch.round(v) if seed is None else torch.floor(v + u)).clamp(-127, 127)
    else:
        v = v.clamp(-448, 448)
        if seed is not None:
            m = v.abs()
            step = (((m.view(torch.int32) >> 23) - 3).clamp_min(127 - 9) << 23).view(torch.float32)
            v = (torch.floor(m / step + u) * step).clamp_max(448) * torch.sign(v)
        v = v.to(torch.float8_e4m3fn).to(torch.float32)
    return v, torch.where(fine, s, torch.full_like(s, 255))


def _values(v, s, features):
    """The values that codes and exponents stand for, (rows, features) in float32."""
    step = torch.where(s == 255, torch.full_like(s, 0x7FC00000), s << 23).view(torch.float32)
    return (v * step[..., None]).reshape(v.shape[0], -1)[:, :features]


def _pack(v, s, features, fmt):
    """Codes and exponents in the layout in which they are kept."""
    rows = v.shape[0]
    width = -(-features // 16) * 16
    codes = v.reshape(rows, -1)[:, :width].to(torch.int8 if fmt == "int8" else torch.float8_e4m3fn)
    panels = -(-features // 128)
    s = torch.nn.functional.pad(s, (0, panels * 4 - s.shape[1]), value=1).reshape(rows, panels, 4)
    s = torch.nn.functional.pad(s, (0, 0, 0, 0, 0, -rows % 64), value=1)
    return codes.contiguous().view(torch.uint8), s.permute(1, 0, 2).to(torch.uint8).contiguous()


def _read(kept, dtype=torch.float32):
    """The values of (codes, scales, features, format), (rows, features)."""
    codes, scales, features, fmt = kept
    rows = codes.shape[0]
    v = codes.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).to(torch.float32)[:, :features].to(dtype)
    s = scales[:, :rows].permute(1, 0, 2).reshape(rows, -1)[:, :-(-features // 32)].to(torch.int32)
    step = torch.where(s == 255, torch.full_like(s, 0x7FC00000), s << 23).view(torch.float32).to(dtype)
    return v * step.repeat_interleave(32, dim=1)[:, :features]


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _activations(rows, features, g, dtype):
    """Activations as they come: normal, a feature in 50 far larger than the rest, tokens of different size."""
    x = torch.randn(rows, features, generator=g, device="cuda")
    x *= torch.where(torch.rand(features, generator=g, device="cuda") < 0.02, 12.0, 0.8)
    x *= torch.exp(0.3 * torch.randn(rows, 1, generator=g, device="cuda"))
    return x.to(_DTYPE[dtype])


def _keep(x, fmt):
    v, s = _quantise(x.float(), fmt)
    codes, scales = _pack(v, s, x.shape[1], fmt)
    return codes, scales, x.shape[1], fmt


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, dt = case["op"], _DTYPE[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    state = {"case": case}
    if op == "save":
        state["x"] = _activations(case["rows"], case["features"], g, case["dtype"])
        state["seed"] = (seed * 0x9E3779B97F4A7C15 + 1) & ((1 << 64) - 1) if case["stochastic"] else None
    elif op == "wgrad":
        state["saved"] = _keep(_activations(case["rows"], case["features"], g, case["dtype"]), case["format"])
        state["dy"] = (normal(case["rows"], case["out"]) * 0.02).to(dt)
        shape = (case["features"], case["out"]) if case["layout"] == "io" else (case["out"], case["features"])
        state["initial"] = normal(*shape).to(_DTYPE[case["out_dtype"]]) if case["initial"] else None
    elif op == "swiglu_fwd":
        both = _activations(case["rows"], 2 * case["features"], g, case["dtype"])  # one projection makes both
        state["gate"], state["up"] = both[:, :case["features"]], both[:, case["features"]:]
    elif op == "swiglu_bwd":
        state["gate"] = _keep(_activations(case["rows"], case["features"], g, case["dtype"]), case["format"])
        state["up"] = _keep(_activations(case["rows"], case["features"], g, case["dtype"]), case["format"])
        state["dh"] = (normal(case["rows"], case["features"]) * 0.02).to(dt)
    else:
        b, t, d = case["batch"], case["seq"], case["features"]
        state["x"] = _activations(b * t, d, g, case["dtype"]).reshape(b, t, d)
        state["branch"] = (_activations(b * t, d, g, case["dtype"]) * 0.5).reshape(b, t, d)
        wide = torch.float32 if dt == torch.float16 else dt
        p = state["param"] = {"kind": case["kind"], "post_norm": case["post_norm"]}
        if case["affine"]:
            p["pre_weight"] = (1 + 0.1 * normal(d)).to(wide)
            if case["kind"] == "layer":
                p["pre_bias"] = (0.1 * normal(d)).to(wide)
            if case["post_norm"]:
                p["post_weight"] = (1 + 0.1 * normal(d)).to(wide)
                if case["kind"] == "layer":
                    p["post_bias"] = (0.1 * normal(d)).to(wide)
        shape = {"none": None, "channel": (d,), "sequence": (b, 1, d), "token": (b, t, 1), "full": (b, t, d)}[case["gate"]]
        if shape is not None:
            p["gate"] = (0.5 + 0.5 * normal(*shape)).to(dt)
            p["gate_activation"] = case["gate_activation"] if case["gate_activation"] != "none" else None
        if case["scale"] == "number":
            p["residual_scale"] = 0.35
        elif case["scale"] == "vector":
            p["residual_scale"] = (0.3 + 0.05 * normal(d)).to(wide)
        if op == "norm_bwd":
            state["dx"] = (normal(b, t, d) * 0.02).to(dt)
            state["dy"] = (normal(b, t, d) * 0.02).to(dt)
            if case["save"] != "none":
                state["x"] = _keep(state["x"].reshape(b * t, d), case["save"])
                state["branch"] = _keep(state["branch"].reshape(b * t, d), case["save"])
    return state


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
_EPS = 1e-6


def _act(gate, name):
    return torch.sigmoid(gate) if name == "sigmoid" else torch.tanh(gate) if name == "tanh" else gate


def _normed(v, kind):
    """(v normalised, its rows' factor)."""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    r = torch.rsqrt((v * v).mean(-1, keepdim=True) + _EPS)
    return v * r, r


def _norm_back(g, n, r, kind):
    """The gradient of the normalised n = (v - mean) * r in v."""
    g = g - n * (g * n).mean(-1, keepdim=True)
    return (g - g.mean(-1, keepdim=True) if kind == "layer" else g) * r


def _norm_fwd(x, b, p):
    n = _normed(b, p["kind"])[0] if p["post_norm"] else b
    if p.get("post_weight") is not None:
        n = n * p["post_weight"].float()
    if p.get("post_bias") is not None:
        n = n + p["post_bias"].float()
    if p.get("gate") is not None:
        n = n * _act(p["gate"].float(), p["gate_activation"])
    s = p.get("residual_scale")
    n = n if s is None else n * (s.float() if isinstance(s, torch.Tensor) else s)
    x = x + n
    y = _normed(x, p["kind"])[0]
    if p.get("pre_weight") is not None:
        y = y * p["pre_weight"].float()
    if p.get("pre_bias") is not None:
        y = y + p["pre_bias"].float()
    return x, y


def _norm_bwd(dx, dy, x, b, p):
    kind, out = p["kind"], {}
    rows = (0, 1)
    nx, rx = _normed(x, kind)
    g = dy
    if p.get("pre_weight") is not None:
        out["pre_weight"] = (dy * nx).sum(rows)
        g = dy * p["pre_weight"].float()
    if p.get("pre_bias") is not None:
        out["pre_bias"] = dy.sum(rows)
    e = dx + _norm_back(g, nx, rx, kind)
    out["x"] = e
    nb, rb = _normed(b, kind) if p["post_norm"] else (b, None)
    n = nb
    if p.get("post_weight") is not None:
        n = n * p["post_weight"].float()
    if p.get("post_bias") is not None:
        n = n + p["post_bias"].float()
    s = p.get("residual_scale")
    f = 1.0 if s is None else s.float() if isinstance(s, torch.Tensor) else s
    gate = _act(p["gate"].float(), p["gate_activation"]) if p.get("gate") is not None else 1.0
    if isinstance(s, torch.Tensor):
        out["residual_scale"] = (e * gate * n).sum(rows)
    if p.get("gate") is not None:
        dg = e * f * n
        shape = (1,) * (3 - p["gate"].dim()) + tuple(p["gate"].shape)
        over = [i for i in (0, 1, 2) if shape[i] == 1]
        dg = (dg.sum(over, keepdim=True) if over else dg).reshape(p["gate"].shape)
        slope = gate * (1 - gate) if p["gate_activation"] == "sigmoid" else 1 - gate * gate if p["gate_activation"] == "tanh" else 1.0
        out["gate"] = dg * slope
    h = e * f * gate
    if p.get("post_bias") is not None:
        out["post_bias"] = h.sum(rows)
    if p.get("post_weight") is not None:
        out["post_weight"] = (h * nb).sum(rows)
        h = h * p["post_weight"].float()
    out["branch"] = _norm_back(h, nb, rb, kind) if p["post_norm"] else h
    return out


def _plain(state):
    case = state["case"]
    op, dt = case["op"], _DTYPE[case["dtype"]]
    most = torch.finfo(dt).max
    if op == "save":
        v, s = _quantise(state["x"].float(), case["format"], state["seed"])
        return _values(v, s, case["features"]).clamp(-most, most).to(dt)
    if op == "wgrad":
        x, dy = _read(state["saved"]), state["dy"].float()
        w = x.t() @ dy if case["layout"] == "io" else dy.t() @ x
        return (w if state["initial"] is None else w + state["initial"].float()).to(_DTYPE[case["out_dtype"]])
    if op == "swiglu_fwd":
        g, u, f = state["gate"].float(), state["up"].float(), case["features"]
        kept = [_values(*_quantise(v, case["format"]), f).clamp(-most, most).to(dt) for v in (g, u)]
        return {"h": (g * torch.sigmoid(g) * u).to(dt), "gate": kept[0], "up": kept[1]}
    if op == "swiglu_bwd":
        g, u, dh = _read(state["gate"]), _read(state["up"]), state["dh"].float()
        s = torch.sigmoid(g)
        h = g * s * u
        return {"gate": (dh * u * s * (1 + g * (1 - s))).to(dt), "up": (dh * g * s).to(dt),
                "h": _values(*_quantise(h, case["format"]), case["features"]).clamp(-most, most).to(dt)}
    p = state["param"]
    if op == "norm_fwd":
        b, t, d = case["batch"], case["seq"], case["features"]
        x, y = _norm_fwd(state["x"].float(), state["branch"].float(), p)
        out = {"x": x.to(dt), "y": y.to(dt)}
        if case["save"] != "none":
            kept = {"x": out["x"], "branch": state["branch"], "y": out["y"]}
            out |= {"saved_" + k: _values(*_quantise(v.reshape(b * t, d).float(), case["save"]), d).clamp(-most, most)
                    .to(dt).reshape(b, t, d) for k, v in kept.items()}
        return out
    shape = state["dx"].shape
    x, b = ((state[k].float() if isinstance(state[k], torch.Tensor) else _read(state[k]).reshape(shape)) for k in ("x", "branch"))
    out = _norm_bwd(state["dx"].float(), state["dy"].float(), x, b, p)
    return {k: v.to(p[k].dtype if k in p else dt) for k, v in out.items()}


def _own(state):
    import rollfast_b200 as rf

    case = state["case"]
    op, dt = case["op"], _DTYPE[case["dtype"]]

    def handle(kept, shape):
        return rf.SavedActivation(kept[0], kept[1], shape, dt, kept[3])

    if op == "save":
        return rf.load_activation(rf.save_activation(state["x"], case["format"], seed=state["seed"]))
    if op == "wgrad":
        saved = handle(state["saved"], (case["rows"], case["features"]))
        return rf.weight_gradient(saved, state["dy"], initial=state["initial"], dtype=_DTYPE[case["out_dtype"]],
                                  layout=case["layout"])
    if op == "swiglu_fwd":
        h, gate, up = rf.swiglu_forward(state["gate"], state["up"], case["format"])
        return {"h": h, "gate": rf.load_activation(gate), "up": rf.load_activation(up)}
    if op == "swiglu_bwd":
        shape = (case["rows"], case["features"])
        gate, up, h = rf.swiglu_backward(state["dh"], handle(state["gate"], shape), handle(state["up"], shape),
                                         save_h=case["format"])
        return {"gate": gate, "up": up, "h": rf.load_activation(h)}
    p = state["param"]
    if op == "norm_fwd":
        r = rf.block_norm_forward(state["x"], state["branch"], eps=_EPS, **p,
                                  save=None if case["save"] == "none" else case["save"])
        out = {"x": r.x, "y": r.y}
        if case["save"] != "none":
            out |= {"saved_x": rf.load_activation(r.saved_x), "saved_branch": rf.load_activation(r.saved_branch),
                    "saved_y": rf.load_activation(r.saved_y)}
        return out
    shape = tuple(state["dx"].shape)
    x, b = (state[k] if isinstance(state[k], torch.Tensor) else handle(state[k], shape) for k in ("x", "branch"))
    r = rf.block_norm_backward(state["dx"], state["dy"], x, b, eps=_EPS, **p)
    return {k: v for k, v in r._asdict().items() if v is not None}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _grid(x, fmt, seed):
    """The 8-bit form's values in 64 bits, from its definition: the step by logarithms, the noise by whole numbers."""
    rows, features = x.shape
    pad = -features % 32
    x = torch.cat([x, x.new_zeros(rows, pad)], 1).reshape(rows, -1, 32)
    most, top = (127.0, 248) if fmt == "int8" else (448.0, 246)
    a = x.abs().amax(-1, keepdim=True)
    m, ex = torch.frexp(a / most)  # a / most = m * 2^ex with m in [0.5, 1)
    e = torch.where(a > 0, ex - (m == 0.5).to(ex.dtype), torch.full_like(ex, -126)).clamp(1 - 127, top - 127)
    step = torch.ldexp(torch.ones_like(a), e)
    if fmt == "e4m3":
        grain = torch.floor(torch.log2((x.abs() / step).clamp_min(2.0 ** -6))) - 3
        step = step * torch.exp2(grain)
    v = (x / step).clamp(-most, most)
    if seed is None:
        v = torch.round(v)
    else:
        u = _noise(rows * features, seed, x.device).double().reshape(rows, features)
        u = torch.cat([u, u.new_zeros(rows, pad)], 1).reshape(x.shape)
        v = torch.floor(v + u) if fmt == "int8" else torch.floor(v.abs() + u) * torch.sign(v)
        v = v.clamp(-127, 127) if fmt == "int8" else v
    return (v * step).reshape(rows, -1)[:, :features]


def _exact_norm(state, case):
    """The forward pass in 64 bits, and its gradients by automatic differentiation."""
    back = case["op"] == "norm_bwd"
    shape = (case["batch"], case["seq"], case["features"])
    leaf = {k: (v.double() if isinstance(v, torch.Tensor) else _read(v, torch.float64).reshape(shape))
            .detach().requires_grad_(back) for k, v in (("x", state["x"]), ("branch", state["branch"]))}
    p = state["param"]
    leaf |= {k: v.double().detach().requires_grad_(back) for k, v in p.items() if isinstance(v, torch.Tensor)}

    def norm(v, weight, bias):
        mean = v.mean(-1, keepdim=True) if p["kind"] == "layer" else 0.0
        v = (v - mean) / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + _EPS)
        v = v * leaf[weight] if weight in leaf else v
        return v + leaf[bias] if bias in leaf else v

    n = norm(leaf["branch"], "post_weight", "post_bias") if p["post_norm"] else leaf["branch"]
    if "gate" in leaf:
        n = n * {"sigmoid": torch.sigmoid, "tanh": torch.tanh, None: torch.clone}[p["gate_activation"]](leaf["gate"])
    s = leaf.get("residual_scale", p.get("residual_scale"))
    # In the backward pass x is the sum already, and the part that the branch adds enters through its gradient alone.
    add = n if s is None else n * s
    if not back:
        total = leaf["x"] + add
        out = {"x": total, "y": norm(total, "pre_weight", "pre_bias")}
        if case["save"] != "none":
            out |= {"saved_" + k: None for k in ("x", "branch", "y")}
        return out
    total = leaf["x"] + add - add.detach()
    y = norm(total, "pre_weight", "pre_bias")
    loss = (total * state["dx"].double()).sum() + (y * state["dy"].double()).sum()
    names = list(leaf)
    return dict(zip(names, torch.autograd.grad(loss, [leaf[k] for k in names])))


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "save":
        return _grid(state["x"].double(), case["format"], state["seed"])
    if op == "wgrad":
        x, dy = _read(state["saved"], torch.float64), state["dy"].double()
        w = torch.einsum("ti,to->io" if case["layout"] == "io" else "ti,to->oi", x, dy)
        return w if state["initial"] is None else w + state["initial"].double()
    if op == "swiglu_fwd":
        g, u = state["gate"].double(), state["up"].double()
        return {"h": g / (1 + torch.exp(-g)) * u, "gate": _grid(g, case["format"], None), "up": _grid(u, case["format"], None)}
    if op == "swiglu_bwd":
        g = _read(state["gate"], torch.float64).requires_grad_()
        u = _read(state["up"], torch.float64).requires_grad_()
        h = g / (1 + torch.exp(-g)) * u
        dg, du = torch.autograd.grad(h, (g, u), state["dh"].double())
        return {"gate": dg, "up": du, "h": None}
    return _exact_norm(state, case)
