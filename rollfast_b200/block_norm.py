"""The norms before and after a block, with its gate, its residual scale and
the residual addition, as one forward and one backward pass.

For a residual stream ``x`` and a block's output ``branch`` (both (..., d)):

    x' = x + residual_scale * act(gate) * N_post(branch)
    y  = N_pre(x')

``y`` is what the next block reads; its parameters are that block's.  N is an
RMS norm (``kind="rms"``) or a LayerNorm (``"layer"``), ``eps`` inside the
root, then weight and bias where given.  Everything is computed in float32 and
each output rounded once; ``y`` comes from the unrounded ``x'``.

Explicit forward / backward pairs (no reference counterpart: there, XLA
differentiates the model).  With ``save``, the forward pass also writes
``x'``, ``branch`` and ``y`` in 8 bits, the first two for the backward pass,
``y`` for the weight gradients of the products that read it.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .activations import (SavedActivation, _format_code, _require_saved, _rows_features, empty_saved, fresh,
                          fresh_bytes, native, on_device, require_same_device, row_strided, stream_of)
from .base import require_cuda, rf_dtype

_KINDS = {"rms": _lib.RF_RMS_NORM, "layer": _lib.RF_LAYER_NORM}
_ACTS = {None: _lib.RF_GATE_IDENTITY, "sigmoid": _lib.RF_GATE_SIGMOID, "tanh": _lib.RF_GATE_TANH}
_PARAMS = ("pre_weight", "pre_bias", "post_weight", "post_bias", "gate", "residual_scale")


class BlockNormOutput(NamedTuple):
    """``x`` (x', or the given x without a branch), ``y`` (None without the
    norm), and with ``save`` each in 8 bits."""

    x: torch.Tensor
    y: torch.Tensor | None
    saved_x: SavedActivation | None
    saved_branch: SavedActivation | None
    saved_y: SavedActivation | None


class BlockNormGrads(NamedTuple):
    """Gradients; None for what was not given (or a number)."""

    x: torch.Tensor
    branch: torch.Tensor | None
    pre_weight: torch.Tensor | None
    pre_bias: torch.Tensor | None
    post_weight: torch.Tensor | None
    post_bias: torch.Tensor | None
    gate: torch.Tensor | None
    residual_scale: torch.Tensor | None


def _gate_layout(gate_shape, shape) -> tuple[int, bool]:
    """(rows that share a row of gates, per channel): the gate broadcasts
    against (..., d), equal to it along the first axes, one along the rest,
    d or one along the last."""
    padded = (1,) * (len(shape) - len(gate_shape)) + tuple(gate_shape)
    lead, gate_lead = shape[:-1], padded[:-1]
    ok = len(padded) == len(shape) and padded[-1] in (1, shape[-1])
    split = 0
    while ok and split < len(lead) and gate_lead[split] == lead[split]:
        split += 1
    if not ok or any(n != 1 for n in gate_lead[split:]):
        raise ValueError(f"gate of shape {tuple(gate_shape)} does not go with arrays of shape {tuple(shape)}: it must "
                         "equal them along the first axes, then be 1, and d or 1 along the last")
    rows = 1
    for n in lead[split:]:
        rows *= n
    return max(rows, 1), padded[-1] == shape[-1]


def _describe(shape, kind, eps, post_norm, params, gate_activation):
    """The checked ctypes description, and the contiguous parameters it points to."""
    if kind not in _KINDS:
        raise ValueError(f"unknown norm kind {kind!r}; expected 'rms' or 'layer'")
    if gate_activation not in _ACTS:
        raise ValueError(f"unknown gate activation {gate_activation!r}; expected None, 'sigmoid' or 'tanh'")
    if not float(eps) >= 0.0:
        raise ValueError(f"eps must be >= 0, got {eps!r}")
    rows, d = _rows_features(tuple(shape), "x")
    p = _lib.RfBlockNorm()
    p.rows, p.features, p.kind, p.post_norm, p.eps, p.scale = rows, d, _KINDS[kind], int(bool(post_norm)), eps, 1.0
    p.gate_rows, p.gate_act = 1, _ACTS[gate_activation]
    keep = {}
    for name in _PARAMS:
        v = params[name]
        if v is None:
            continue
        if name == "residual_scale" and not isinstance(v, torch.Tensor):
            p.scale = float(v)
            continue
        require_cuda(v, name)
        dt = rf_dtype(v)
        if name == "gate":
            p.gate_rows, per_channel = _gate_layout(v.shape, shape)
            p.gate_per_channel = int(per_channel)
        elif name == "residual_scale" and v.numel() == 1 and v.ndim <= 1:
            p.scale_per_channel = int(d == 1)
        elif tuple(v.shape) != (d,):
            raise ValueError(f"{name} must have shape ({d},), got {tuple(v.shape)}")
        elif name == "residual_scale":
            p.scale_per_channel = 1
        if name.startswith("post_") and not post_norm:
            raise ValueError(f"{name} needs post_norm=True")
        keep[name] = v.contiguous()
        field = getattr(p, name)
        field.value, field.dtype = keep[name].data_ptr(), dt
    return p, keep


def _refuse_unused(branch, given: dict, pre_norm: bool = True) -> None:
    """Parameters of a part that the call leaves out: without an error, a
    forgotten branch or norm would go unnoticed."""
    if branch is None:
        extra = [n for n in ("post_weight", "post_bias", "gate") if given[n] is not None]
        if isinstance(given["residual_scale"], torch.Tensor):
            extra.append("residual_scale")
        if extra:
            raise ValueError(f"{', '.join(extra)} given without a branch")
    extra = [n for n in ("pre_weight", "pre_bias") if given[n] is not None]
    if extra and not pre_norm:
        raise ValueError(f"{', '.join(extra)} given with pre_norm=False")


def _rows(t, what: str, shape):
    """(RfRows, what must stay alive)"""
    if isinstance(t, SavedActivation):
        _require_saved(t, what)
        if t.shape != shape:
            raise ValueError(f"{what} must have shape {shape}, got {t.shape}")
        s = t._native()
        return _lib.RfRows(None, 0, 0, ctypes.pointer(s)), (t, s)
    require_cuda(t, what)
    if tuple(t.shape) != shape:
        raise ValueError(f"{what} must have shape {shape}, got {tuple(t.shape)}")
    dt = rf_dtype(t)
    t, ld = row_strided(t)
    return _lib.RfRows(t.data_ptr(), ld, dt, None), t


def _like(t, others, device):
    """An array for the gradient of ``t``, a tensor or a saved activation."""
    if isinstance(t, torch.Tensor):
        return fresh(t)
    for o in others:  # of the same shape
        if o is not None and o.dtype == t.dtype:
            return fresh(o)
    return torch.empty(t.shape, dtype=t.dtype, device=device)


def block_norm_forward(x: torch.Tensor, branch: torch.Tensor | None = None, *, kind: str = "rms", eps: float = 1e-6,
                       post_norm: bool = True, pre_norm: bool = True, pre_weight: torch.Tensor | None = None,
                       pre_bias: torch.Tensor | None = None, post_weight: torch.Tensor | None = None,
                       post_bias: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                       gate_activation: str | None = None, residual_scale=None,
                       save: str | None = None) -> BlockNormOutput:
    """``x' = x + residual_scale * act(gate) * N_post(branch)``, ``y = N_pre(x')``.

    Without ``branch`` (before the first block) ``y = N_pre(x)``; with
    ``pre_norm=False`` (after the last) there is no ``y``; tensors of the part
    that is left out are refused.  With ``post_norm=False`` the branch is added
    as it is.  ``gate`` broadcasts against ``x``: equal to it along the first
    axes, 1 along the rest, d or 1 along the last -- (d,), (batch, 1, d),
    (batch, tokens, 1), ``x``'s own shape.  ``residual_scale``: a number, (d,)
    or one element.  x' has ``x``'s dtype, ``y`` the branch's (``x``'s without
    one).  At most 16384 features."""
    require_cuda(x, "x")
    rf_dtype(x)
    shape = tuple(x.shape)
    given = dict(pre_weight=pre_weight, pre_bias=pre_bias, post_weight=post_weight, post_bias=post_bias, gate=gate,
                 residual_scale=residual_scale)
    _refuse_unused(branch, given, pre_norm)
    p, keep = _describe(shape, kind, eps, post_norm, given, gate_activation)
    if save is not None:
        _format_code(save)
    if branch is not None:
        require_cuda(branch, "branch")
    require_same_device(x.device, branch=branch, **keep)
    device = x.device
    lib = _lib.load()
    with on_device(device):
        cx, alive_x = _rows(x, "x", shape)
        cb, alive_b = (None, None) if branch is None else _rows(branch, "branch", shape)
        out = fresh(x) if branch is not None else x
        y = fresh(x if branch is None else branch) if pre_norm else None
        saved = [None if save is None or t is None else empty_saved(shape, t.dtype, save, device)
                 for t in (out, branch, y)]
        co = None if branch is None else _rows(out, "x", shape)[0]
        cy = None if y is None else _rows(y, "y", shape)[0]
        _lib.check(lib.rf_block_norm_forward(p, cx, cb, co, cy, *(native(s) for s in saved), stream_of(device)))
    del alive_x, alive_b
    return BlockNormOutput(out, y, *saved)


def block_norm_backward(grad_x: torch.Tensor | None, grad_y: torch.Tensor | None, x, branch=None, *,
                        kind: str = "rms", eps: float = 1e-6, post_norm: bool = True,
                        pre_weight: torch.Tensor | None = None, pre_bias: torch.Tensor | None = None,
                        post_weight: torch.Tensor | None = None, post_bias: torch.Tensor | None = None,
                        gate: torch.Tensor | None = None, gate_activation: str | None = None,
                        residual_scale=None) -> BlockNormGrads:
    """Gradients of ``block_norm_forward`` from those of x' (``grad_x``) and
    ``y`` (``grad_y``); either may be None, for zeros.

    ``x`` is x' (the forward pass's output) and ``branch`` the block's output,
    each an array or a ``SavedActivation``; row statistics are formed again
    from them.  The other arguments are the forward pass's.  The gradient of
    ``x`` has ``x``'s dtype, the branch's the branch's, a parameter's the
    parameter's.  Sums over rows are formed in float32 in a fixed order."""
    if grad_x is None and grad_y is None:
        raise ValueError("block_norm_backward needs grad_x or grad_y")
    if x is None:
        raise ValueError("block_norm_backward needs x")
    shape = tuple(x.shape)
    given = dict(pre_weight=pre_weight, pre_bias=pre_bias, post_weight=post_weight, post_bias=post_bias, gate=gate,
                 residual_scale=residual_scale)
    p, keep = _describe(shape, kind, eps, post_norm, given, gate_activation)
    _refuse_unused(branch, given)
    device = x.device
    for name, t in (("grad_x", grad_x), ("grad_y", grad_y)):
        if t is not None:
            require_cuda(t, name)
    require_same_device(device, grad_x=grad_x, grad_y=grad_y, branch=branch, **keep)
    lib = _lib.load()
    with on_device(device):
        args, alive = [], []
        for name, t in (("grad_x", grad_x), ("grad_y", grad_y), ("x", x), ("branch", branch)):
            c, a = (None, None) if t is None else _rows(t, name, shape)
            args.append(c)
            alive.append(a)
        empty = p.rows == 0
        make = torch.zeros_like if empty else torch.empty_like
        out_x = _like(x, (grad_x, grad_y), device)
        out_b = None if branch is None else _like(branch, (grad_y, grad_x), device)
        grads = {n: make(t) for n, t in keep.items()}
        if not empty:
            for n, t in grads.items():
                getattr(p, n).grad = t.data_ptr()
            args.append(_rows(out_x, "x", shape)[0])
            args.append(None if out_b is None else _rows(out_b, "branch", shape)[0])
            nbytes = ctypes.c_size_t()
            _lib.check(lib.rf_block_norm_workspace_size(p, ctypes.byref(nbytes)))
            ws = fresh_bytes(nbytes.value, device) if nbytes.value else None
            _lib.check(lib.rf_block_norm_backward(p, *args, None if ws is None else ws.data_ptr(), nbytes.value,
                                                  stream_of(device)))
    del alive
    return BlockNormGrads(out_x, out_b, *(grads.get(n) for n in BlockNormGrads._fields[2:]))


__all__ = ["BlockNormGrads", "BlockNormOutput", "block_norm_backward", "block_norm_forward"]
