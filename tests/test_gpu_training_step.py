"""The training-step operators together, as a user runs them: one feed-forward
block between its norms, forward and backward over 8-bit activations, its
weight gradients into ``muon`` and its vectors into the AdamW branch."""

import numpy as np
import pytest
import torch

from oracle import training_np as T

pytestmark = pytest.mark.gpu

EPS = 1e-6


def _params(d, f, dt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def mat(a, b):
        return (torch.randn(a, b, generator=g, device="cuda") / a ** 0.5).to(dt)

    def vec(mean):
        return mean + 0.1 * torch.randn(d, generator=g, device="cuda")

    return {"gate_up": mat(d, 2 * f), "down": mat(f, d), "pre": vec(1.0), "post": vec(1.0), "gate": vec(0.5),
            "scale": vec(0.3), "next": vec(1.0)}


def forward(p, x, fmt):
    """x -> (x', y, what the backward pass keeps): no activation is kept in 16 bits."""
    import rollfast_b200 as rf

    f = p["down"].shape[0]
    first = rf.block_norm_forward(x, eps=EPS, pre_weight=p["pre"], save=fmt)
    both = first.y @ p["gate_up"]
    h, sg, su = rf.swiglu_forward(both[..., :f], both[..., f:], fmt)
    branch = h @ p["down"]
    last = rf.block_norm_forward(x, branch, eps=EPS, post_weight=p["post"], gate=p["gate"], gate_activation="sigmoid",
                                 residual_scale=p["scale"], pre_weight=p["next"], save=fmt)
    return last.x, last.y, (first.saved_x, first.saved_y, sg, su, last.saved_x, last.saved_branch)


def backward(p, kept, dx, dy, fmt):
    import rollfast_b200 as rf

    sx, sy, sg, su, sx2, sb = kept
    f = p["down"].shape[0]
    g2 = rf.block_norm_backward(dx, dy, sx2, sb, eps=EPS, post_weight=p["post"], gate=p["gate"],
                                gate_activation="sigmoid", residual_scale=p["scale"], pre_weight=p["next"])
    dh = g2.branch @ p["down"].t()
    dboth = torch.empty(*dh.shape[:-1], 2 * f, dtype=dh.dtype, device=dh.device)
    _, _, sh = rf.swiglu_backward(dh, sg, su, save_h=fmt, grad_gate=dboth[..., :f], grad_up=dboth[..., f:])
    dn = dboth @ p["gate_up"].t()
    g1 = rf.block_norm_backward(g2.x, dn, sx, eps=EPS, pre_weight=p["pre"])
    return g1.x, {"gate_up": rf.weight_gradient(sy, dboth), "down": rf.weight_gradient(sh, g2.branch),
                  "pre": g1.pre_weight, "post": g2.post_weight, "gate": g2.gate, "scale": g2.residual_scale,
                  "next": g2.pre_weight}


def exact(p, x, dx, dy):
    """The step's gradients in 64 bits from the unrounded forward pass."""
    q = {k: v.double().cpu().numpy() for k, v in p.items()}
    x, dx, dy = (t.double().cpu().numpy() for t in (x, dx, dy))
    f = q["down"].shape[0]
    n, r = T.normalised(x, "rms", EPS)
    y = n * q["pre"]
    both = y @ q["gate_up"]
    g, u = both[..., :f], both[..., f:]
    h = T.swiglu(g, u)
    b = h @ q["down"]
    par = {"post_weight": q["post"], "gate": q["gate"], "residual_scale": q["scale"], "pre_weight": q["next"]}
    kw = dict(gate_activation="sigmoid", eps=EPS)
    out = T.block_norm_grads(dx, dy, T.block_norm(x, b, par, **kw)[0], b, par, **kw)
    dh = out["branch"] @ q["down"].T
    dboth = np.concatenate(T.swiglu_grads(dh, g, u), -1)
    first = T.block_norm_grads(out["x"], dboth @ q["gate_up"].T, x, None, {"pre_weight": q["pre"]}, eps=EPS)
    return first["x"], {"gate_up": T.weight_gradient(y, dboth), "down": T.weight_gradient(h, out["branch"]),
                        "pre": first["pre_weight"], "post": out["post_weight"], "gate": out["gate"],
                        "scale": out["residual_scale"], "next": out["pre_weight"]}


@pytest.mark.parametrize("fmt,dt", [("int8", torch.float32), ("int8", torch.bfloat16), ("e4m3", torch.float32)])
@pytest.mark.parametrize("shape", [(2, 150, 192, 320), (1, 33, 136, 72)], ids=str)
def test_step_gradients(fmt, dt, shape):
    """Against 64 bits without any 8-bit form: what is off is the activations'
    rounding.  int8: a code is off by at most half of 2/127 of its block's
    largest magnitude, uniform over the steps, so about 2 max / (127 sqrt 12)
    in the mean square, for blocks of 32 normal values (max about 2.1 times
    the root mean square) at most 2^-6.9 of the activation.  e4m3: at most half
    of 2^-3 of each value, in the mean square 2^-3 / sqrt 12 = 2^-4.8.  At
    most four saved activations enter a gradient, each to first order with a
    weight of at most 2 (a product of two rounded factors); bfloat16 rounding
    of the arrays between (2^-9 each) is small beside that.  So int8 stays
    within 8 * 2^-6.9 and e4m3 within 8 * 2^-4.8 of a gradient's norm."""
    b, t, d, f = shape
    p = _params(d, f, dt)
    g = torch.Generator(device="cuda").manual_seed(5)
    x, dx, dy = (torch.randn(b, t, d, generator=g, device="cuda").to(dt) for _ in range(3))
    _, _, kept = forward(p, x, fmt)
    dx0, grads = backward(p, kept, dx, dy, fmt)
    wx, want = exact(p, x, dx, dy)
    most = 8 * 2.0 ** (-6.9 if fmt == "int8" else -4.8)
    for name, got, w in [("x", dx0, wx)] + [(k, grads[k], want[k]) for k in want]:
        err = np.linalg.norm(got.double().cpu().numpy() - w) / np.linalg.norm(w)
        assert got.shape == w.shape and err <= most, (name, err)


def test_step_into_muon_and_a_captured_pass():
    """The gradients go into muon(...) as they are; a captured forward and
    backward pass gives the eager bits for new inputs."""
    import rollfast_b200 as rf

    dt = torch.bfloat16
    p = _params(192, 320, dt)
    x, dx, dy = (torch.randn(2, 150, 192, device="cuda").to(dt) for _ in range(3))
    tx = rf.muon(learning_rate=0.02, weight_decay=0.01)
    state = tx.init(p)

    def step():
        y0, y1, kept = forward(p, x, "int8")
        return y0, y1, *backward(p, kept, dx, dy, "int8")[1].values()

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        captured = step()
    for _ in range(2):
        x.copy_(torch.randn_like(x))
        dy.copy_(torch.randn_like(dy))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)
        _, _, kept = forward(p, x, "int8")
        grads = backward(p, kept, dx, dy, "int8")[1]
        updates, state = tx.update(grads, state, p)
        new = rf.apply_updates(p, updates, key=3)
        for k in p:
            assert new[k].shape == p[k].shape and new[k].isfinite().all() and not torch.equal(new[k], p[k])
            p[k].copy_(new[k])


def test_another_device_is_refused_or_used():
    import rollfast_b200 as rf

    x = torch.randn(4, 64, device="cuda")
    saved = rf.save_activation(x)
    with pytest.raises(ValueError):
        rf.weight_gradient(saved, torch.randn(4, 8))
    with pytest.raises(ValueError):
        rf.block_norm_forward(x, pre_weight=torch.ones(64))
