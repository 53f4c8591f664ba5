"""Activations kept in 8 bits between the forward and the backward pass, and
the backward work that reads them: the weight gradients that ``muon`` takes,
and a SwiGLU.

Explicit forward / backward pairs, as a custom derivative rule binds them (no
reference counterpart: there, XLA differentiates the model).  Arrays are CUDA
``torch.Tensor``s with features along the last axis; the other axes are rows.
Row-strided views (one half of a fused projection) are read in place, other
layouts are copied.  Calls are queued on the current stream of the arrays'
device and return at once; results carry no autograd history.

The 8-bit form cuts a row into blocks of 32 features: 32 codes (``"int8"`` or
``"e4m3"``) and a power-of-two step as small as the block's largest magnitude
allows.  int8 has steps of 1/127 to 2/127 of a block's largest magnitude, e4m3
a relative error of at most 2^-4; both take 1.03 bytes per element.  With a
``seed``, rounding is stochastic, as in ``apply_updates``: a value between two
codes goes to the upper one (e4m3: the larger in magnitude) with the
probability of its distance from the other, rounded down to 2^-16.  So the mean
of a code is the value to within 2^-16 of a step, and weight gradients, which
are linear in it, are unbiased to that.  A block with an infinity or a NaN
reads as NaN throughout.
"""

from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _lib
from .base import require_cuda, rf_dtype

_LAYOUTS = {"io": _lib.RF_IN_OUT, "oi": _lib.RF_OUT_IN}


class SavedActivation:
    """An activation in 8 bits: ``codes`` (rows, features rounded up to 16)
    and ``scales`` (panels of 128 features, rows rounded up to 64, 4), both
    contiguous ``uint8``; the ``shape`` and ``dtype`` of the original, and the
    ``format``.  value = code * 2^(scale - 127), a scale of 255 meaning NaN;
    the scale of feature f is ``scales[f // 128, row, f % 128 // 32]``."""

    __slots__ = ("_codes", "_scales", "_buffer", "shape", "dtype", "format", "rows", "features")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape, dtype: torch.dtype, format: str):
        _format_code(format)
        shape = tuple(int(n) for n in shape)
        rows, features = _rows_features(shape, "a saved activation")
        want = [((rows, _up(features, 16)), codes, "codes"), ((-(-features // 128), _up(rows, 64), 4), scales, "scales")]
        for expected, t, name in want:
            if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8 or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous uint8 tensor")
            if tuple(t.shape) != expected:
                raise ValueError(f"{name} of an activation of shape {shape} must have shape {expected}, "
                                 f"got {tuple(t.shape)}")
        if codes.device != scales.device:
            raise ValueError("codes and scales must be on one device")
        self._codes, self._scales, self._buffer = codes, scales, None
        self.shape, self.dtype, self.format, self.rows, self.features = shape, dtype, format, rows, features

    @classmethod
    def _empty(cls, shape, dtype, format, device) -> "SavedActivation":
        """One allocation for codes and scales; their tensors are made when
        someone asks for them."""
        self = object.__new__(cls)
        self.rows, self.features = rows, features = _rows_features(shape, "a saved activation")
        self.shape, self.dtype, self.format = shape, dtype, format
        self._codes = self._scales = None
        self._buffer = fresh_bytes(_up(rows * _up(features, 16), 256) + -(-features // 128) * _up(rows, 64) * 4, device)
        return self

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            ld = _up(self.features, 16)
            self._codes = self._buffer[:self.rows * ld].view(self.rows, ld)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._scales = self._buffer[_up(self.rows * _up(self.features, 16), 256):].view(
                -(-self.features // 128), _up(self.rows, 64), 4)
        return self._scales

    def _native(self) -> _lib.RfSavedActivation:
        ld, code = _up(self.features, 16), _lib.FORMAT8_CODES[self.format]
        if self._buffer is not None:
            codes = self._buffer.data_ptr()
            scales = codes + _up(self.rows * ld, 256)
        else:
            codes, scales = self._codes.data_ptr(), self._scales.data_ptr()
        return _lib.RfSavedActivation(codes, scales, self.rows, self.features, ld, _up(self.rows, 64), code)

    @property
    def device(self) -> torch.device:
        return (self._codes if self._buffer is None else self._buffer).device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def __repr__(self) -> str:
        return f"SavedActivation(shape={self.shape}, dtype={self.dtype}, format={self.format!r})"


def _up(a: int, b: int) -> int:
    return -(-a // b) * b


def _format_code(format: str) -> int:
    try:
        return _lib.FORMAT8_CODES[format]
    except (KeyError, TypeError):
        raise ValueError(f"unknown 8-bit format {format!r}; expected 'int8' or 'e4m3'") from None


def _rows_features(shape, what: str) -> tuple[int, int]:
    if not shape or shape[-1] < 1:
        raise ValueError(f"{what} needs at least one feature along its last axis, got shape {tuple(shape)}")
    rows = 1
    for n in shape[:-1]:
        rows *= n
    return rows, shape[-1]


def row_strided(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """``t`` as rows along all axes but the last, one stride apart: itself
    where its strides allow, else a contiguous copy; and that stride."""
    d = t.shape[-1]
    if t.is_contiguous():
        return t, d
    if t.stride(-1) == 1 or d == 1:
        ld = expected = None
        for n, s in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if n == 1:
                continue
            if ld is None:
                ld = expected = s
            elif s != expected:
                break
            expected = expected * n
        else:
            if ld is None or ld >= d:
                return t, d if ld is None else ld
    return t.contiguous(), d


def _out_rows(t: torch.Tensor, what: str) -> int:
    """Row stride of an output, which cannot be copied."""
    same, ld = row_strided(t)
    if same is not t:
        raise ValueError(f"{what} must have contiguous features and evenly strided rows")
    return ld


_here = contextlib.nullcontext()


def on_device(device: torch.device):
    """A launch must come from the arrays' device; switching costs more than
    the check that it is current already."""
    return _here if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


def stream_of(device: torch.device) -> int:
    """Handle of the current stream, without a Stream object: that takes
    microseconds, as much as a small call's launch."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def fresh(like: torch.Tensor) -> torch.Tensor:
    """A contiguous array of ``like``'s shape and type, by the quickest way
    that makes one: of a small call's time, half went into ``torch.empty``."""
    return torch.empty_like(like) if like.is_contiguous() else torch.empty(like.shape, dtype=like.dtype,
                                                                           device=like.device)


def fresh_bytes(n: int, device: torch.device) -> torch.Tensor:
    return torch.empty_strided((n,), (1,), dtype=torch.uint8, device=device)


def require_same_device(device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, expected {device}")


def native(saved: SavedActivation | None):
    """The ctypes form, or None."""
    return None if saved is None else saved._native()


def empty_saved(shape, dtype: torch.dtype, format: str, device: torch.device) -> SavedActivation:
    _format_code(format)
    return SavedActivation._empty(tuple(shape), dtype, format, device)


def _require_saved(saved, what: str) -> None:
    if not isinstance(saved, SavedActivation):
        raise ValueError(f"{what} must be a SavedActivation, got {type(saved).__name__}")
    if saved.device.type != "cuda":
        require_cuda(saved.codes, what)


def _check_seed(seed) -> int:
    if isinstance(seed, bool) or not isinstance(seed, int) or not 0 <= seed < 1 << 64:
        raise ValueError(f"seed must be an integer in [0, 2**64), got {seed!r}")
    return seed


def save_activation(x: torch.Tensor, format: str = "int8", *, seed: int | None = None) -> SavedActivation:
    """``x`` (..., features; float32, bfloat16 or float16) in 8 bits, to
    nearest even, or stochastically with the SplitMix64 noise of ``seed``
    (16 bits per element, in element order).  A call captured into a CUDA
    graph keeps its seed over replays."""
    require_cuda(x, "x")
    dt = rf_dtype(x)
    _rows_features(tuple(x.shape), "x")
    stochastic = seed is not None
    seed = _check_seed(seed) if stochastic else 0
    lib = _lib.load()
    with on_device(x.device):
        saved = empty_saved(x.shape, x.dtype, format, x.device)
        x, ld = row_strided(x)
        _lib.check(lib.rf_save_activation(x.data_ptr(), ld, dt, native(saved), int(stochastic), seed,
                                          stream_of(x.device)))
    return saved


def load_activation(saved: SavedActivation, *, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The values that ``saved`` stands for, in ``dtype`` (the original's by
    default): exact in float32 and bfloat16 but for subnormals; float16
    saturates at 65504."""
    _require_saved(saved, "saved")
    lib = _lib.load()
    with on_device(saved.device):
        out = torch.empty(saved.shape, dtype=dtype or saved.dtype, device=saved.device)
        _lib.check(lib.rf_load_activation(native(saved), out.data_ptr(), saved.features, rf_dtype(out),
                                          stream_of(saved.device)))
    return out


def weight_gradient(saved: SavedActivation, grad_output: torch.Tensor, *, initial: torch.Tensor | None = None,
                    out: torch.Tensor | None = None, dtype: torch.dtype | None = None,
                    layout: str = "io") -> torch.Tensor:
    """Gradient of W in ``y = x @ W`` from the saved ``x`` (..., in) and the
    gradient of ``y`` (..., out): the sum over all rows of their outer
    products, plus ``initial``.

    ``layout``: ``"io"`` gives (in, out), the layout of ``muon``'s leaves;
    ``"oi"`` the transpose.  ``initial`` (the result's shape) adds an earlier
    gradient before the only rounding; with ``out=initial`` the sum is
    accumulated in place, otherwise ``out`` must not overlap an input.
    ``dtype``: float32 by default, or that of ``out`` or ``initial``.

    The sum is held in float32.  The saved values enter the tensor cores
    exactly, and so does a bfloat16 gradient; a float16 or float32 gradient is
    split into two or three bfloat16 terms that add up to it (but for parts
    below 2^-133), at two or three times the work.  Equal operands give equal
    bits.  While it runs, the call holds a workspace: the activation once in
    bfloat16; the terms of a gradient that is not bfloat16, or one copy of a
    bfloat16 gradient whose rows do not start on 16-byte boundaries; and, where
    the sum over tokens is split, the float32 parts of at most 73 tiles of
    256 x 256."""
    _require_saved(saved, "saved")
    require_cuda(grad_output, "grad_output")
    try:
        code = _LAYOUTS[layout]
    except (KeyError, TypeError):
        raise ValueError(f"unknown layout {layout!r}; expected 'io' or 'oi'") from None
    if tuple(grad_output.shape[:-1]) != saved.shape[:-1] or grad_output.ndim != len(saved.shape):
        raise ValueError(f"grad_output of shape {tuple(grad_output.shape)} does not go with an activation of shape "
                         f"{saved.shape}")
    _, n_out = _rows_features(tuple(grad_output.shape), "grad_output")
    gdt = rf_dtype(grad_output)
    device = saved.device
    require_same_device(device, grad_output=grad_output, initial=initial, out=out)
    shape = (saved.features, n_out) if layout == "io" else (n_out, saved.features)
    given = out.dtype if out is not None else initial.dtype if initial is not None else dtype or torch.float32
    for name, t in (("initial", initial), ("out", out)):
        if t is None:
            continue
        require_cuda(t, name)
        if tuple(t.shape) != shape:
            raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
        if t.dtype != given or (dtype is not None and t.dtype != dtype):
            raise ValueError(f"{name} has dtype {t.dtype}, expected {dtype or given}")
    lib = _lib.load()
    with on_device(device):
        if out is None:
            out = torch.empty(shape, dtype=given, device=device)
        ld_out = _out_rows(out, "out")
        if initial is not None and initial.stride() != out.stride():
            same, ld = row_strided(initial)
            if ld != ld_out:
                same = torch.empty_strided(out.shape, out.stride(), dtype=out.dtype, device=device).copy_(initial)
            initial = same
        grad_output, ldg = row_strided(grad_output)
        nbytes = ctypes.c_size_t()
        _lib.check(lib.rf_weight_gradient_workspace_size(saved.rows, saved.features, n_out, grad_output.data_ptr(), ldg,
                                                         gdt, ctypes.byref(nbytes)))
        # Allocated per call: a cached buffer would be shared by CUDA graphs
        # that are captured on one stream and replayed on two.
        ws = fresh_bytes(nbytes.value, device) if nbytes.value else None
        _lib.check(lib.rf_weight_gradient(native(saved), grad_output.data_ptr(), ldg, gdt, n_out, code,
                                          None if initial is None else initial.data_ptr(), out.data_ptr(), ld_out,
                                          rf_dtype(out), None if ws is None else ws.data_ptr(), nbytes.value,
                                          stream_of(device)))
    return out


def swiglu_forward(gate: torch.Tensor, up: torch.Tensor, format: str | None = "int8"):
    """``h = silu(gate) * up``, and both inputs saved in 8 bits for
    ``swiglu_backward``: ``(h, saved_gate, saved_up)``.  ``format=None`` saves
    nothing (the two are None)."""
    require_cuda(gate, "gate")
    require_cuda(up, "up")
    if gate.shape != up.shape or gate.dtype != up.dtype:
        raise ValueError(f"gate and up must agree in shape and dtype, got {tuple(gate.shape)} {gate.dtype} and "
                         f"{tuple(up.shape)} {up.dtype}")
    dt = rf_dtype(gate)
    rows, features = _rows_features(tuple(gate.shape), "gate")
    require_same_device(gate.device, up=up)
    device = gate.device
    lib = _lib.load()
    with on_device(device):
        h = fresh(gate)
        sg = su = None
        if format is not None:
            sg = empty_saved(gate.shape, gate.dtype, format, device)
            su = empty_saved(gate.shape, gate.dtype, format, device)
        gate, ldg = row_strided(gate)
        up, ldu = row_strided(up)
        _lib.check(lib.rf_swiglu_forward(gate.data_ptr(), ldg, up.data_ptr(), ldu, h.data_ptr(), features, dt, rows,
                                         features, native(sg), native(su), stream_of(device)))
    return h, sg, su


def swiglu_backward(grad_h: torch.Tensor, saved_gate: SavedActivation, saved_up: SavedActivation, *,
                    save_h: str | None = None, grad_gate: torch.Tensor | None = None,
                    grad_up: torch.Tensor | None = None):
    """Gradients of ``swiglu_forward`` at the saved inputs, in ``grad_h``'s
    dtype, and with ``save_h`` (a format) ``h`` formed again from them in
    float32 and saved, for the weight gradient of the product that reads it --
    so the forward pass need not keep it: ``(grad_gate, grad_up, saved_h)``.
    ``grad_gate`` / ``grad_up``: arrays to write to (row-strided: the halves
    of a fused projection's gradient); one of them may be ``grad_h`` itself."""
    require_cuda(grad_h, "grad_h")
    _require_saved(saved_gate, "saved_gate")
    _require_saved(saved_up, "saved_up")
    dt = rf_dtype(grad_h)
    shape = tuple(grad_h.shape)
    if saved_gate.shape != shape or saved_up.shape != shape:
        raise ValueError(f"grad_h of shape {shape} does not go with saved activations of shapes {saved_gate.shape} "
                         f"and {saved_up.shape}")
    device = grad_h.device
    require_same_device(device, saved_gate=saved_gate, saved_up=saved_up, grad_gate=grad_gate, grad_up=grad_up)
    for name, t in (("grad_gate", grad_gate), ("grad_up", grad_up)):
        if t is not None and (tuple(t.shape) != shape or t.dtype != grad_h.dtype):
            raise ValueError(f"{name} must have grad_h's shape {shape} and dtype {grad_h.dtype}")
    if grad_gate is not None and grad_up is not None and grad_gate.numel() and grad_gate.data_ptr() == grad_up.data_ptr():
        raise ValueError("grad_gate and grad_up must be two arrays")
    lib = _lib.load()
    with on_device(device):
        if grad_gate is None:
            grad_gate = fresh(grad_h)
        if grad_up is None:
            grad_up = fresh(grad_h)
        ldg, ldu = _out_rows(grad_gate, "grad_gate"), _out_rows(grad_up, "grad_up")
        saved_h = None if save_h is None else empty_saved(shape, saved_gate.dtype, save_h, device)
        grad_h, ldh = row_strided(grad_h)
        _lib.check(lib.rf_swiglu_backward(grad_h.data_ptr(), ldh, native(saved_gate), native(saved_up),
                                          grad_gate.data_ptr(), ldg, grad_up.data_ptr(), ldu, dt, native(saved_h),
                                          stream_of(device)))
    return grad_gate, grad_up, saved_h


__all__ = ["SavedActivation", "load_activation", "save_activation", "swiglu_backward", "swiglu_forward",
           "weight_gradient"]
