"""The gated linear recurrence: the scan over a sequence, with its gradients, and the step of one sample.

    z = (f | v | o) along the channels
    h_t = sigmoid(f_t) h_{t-1} + (1 - sigmoid(f_t)) v_t        y_t = h_t sigmoid(o_t)        (no output gate: y = h)

The recurrent counterpart of the gated convolution of ``modules.ResidualConv1dGLU`` (reference modules.py:112-169): its whole past is
one state of C float32 numbers instead of a history ring.  All arithmetic happens in libwnv_hip.so (``wnv_recurrence_*`` in
include/wnv.h); there is no CPU path.
"""
from __future__ import annotations

import ctypes as C
from functools import lru_cache
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _lib
from ._lib import DTYPE, RecurrenceArgs, check
from .engine import _raw_stream, refuse_tangents, require_gpu_tensor

__all__ = ["gated_recurrence", "gated_recurrence_step"]

_DTYPES = {getattr(torch, name): code for name, code in DTYPE.items()}


def _dtype(z: torch.Tensor) -> int:
    code = _DTYPES.get(z.dtype)
    if code is None:
        raise TypeError(f"z is {z.dtype}: float32, bfloat16 and float16 are implemented")
    return code


def _state(h: torch.Tensor, name: str, B: int, n: int, z: torch.Tensor) -> torch.Tensor:
    if h.shape != (B, n):
        raise ValueError(f"{name} is {tuple(h.shape)}, expected {(B, n)}")
    if h.dtype != torch.float32:
        raise TypeError(f"{name} is {h.dtype}: the state is float32")
    if h.get_device() != z.get_device():
        raise ValueError(f"{name} lives on {h.device}, z on {z.device}")
    return h


def _map(m: torch.Tensor, name: str, shape: Tuple[int, ...], z: torch.Tensor) -> torch.Tensor:
    if m.shape != shape:
        raise ValueError(f"{name} is {tuple(m.shape)}, expected {shape}")
    if m.get_device() != z.get_device():
        raise ValueError(f"{name} lives on {m.device}, z on {z.device}")
    if m.dtype == torch.int64:
        m = m.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    elif m.dtype != torch.int32:
        raise TypeError(f"{name} is {m.dtype}: int32 or int64")
    return m.contiguous()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with its last dimension contiguous: a copy only where it is not, or where steps lie 2^20 elements and more apart."""
    n = t.shape[-1]
    return t if (t.stride(-1) == 1 or n == 1) and (t.dim() < 3 or t.stride(1) < max(n + 1, 1 << 20)) else t.contiguous()


@lru_cache(maxsize=256)
def _sizes(B: int, T: int, n: int, gates: int, code: int) -> Tuple[int, int]:
    """Bytes of (saved, workspace), which go by the shape alone."""
    lib = _lib.lib()
    saved = lib.wnv_recurrence_saved_bytes(B, T, n, gates, code)
    if saved < 0:
        raise ValueError(lib.wnv_last_error().decode())
    return saved, lib.wnv_recurrence_workspace_bytes(B, T, n, gates, code)


# The two calls below write their arguments out without helpers: short sequences are the host's time (5 x 15 x 16 forward and backward 104
# us, through helpers 108).  The workspace is of the stream that runs the call: torch's allocator hands it out again behind the call's
# own work only.
def _forward(z, h0, gates, lengths, seg_start, keep: bool):
    B, T, n = z.shape
    n //= gates
    code, dev, index = _DTYPES[z.dtype], z.device, z.get_device()
    saved_bytes, ws_bytes = _sizes(B, T, n, gates, code)
    y = z.new_empty((B, T, n))
    h_last = torch.empty((B, n), dtype=torch.float32, device=dev)
    saved = torch.empty(saved_bytes, dtype=torch.uint8, device=dev) if keep else None
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    zb, zt, _ = z.stride()
    a = RecurrenceArgs(B, n, T, gates, code, z.data_ptr(), zb, zt, None if h0 is None else h0.data_ptr(), 0 if h0 is None else h0.stride(0),
                       None if lengths is None else lengths.data_ptr(), None if seg_start is None else seg_start.data_ptr(), y.data_ptr(),
                       h_last.data_ptr(), None if saved is None else saved.data_ptr(), None if ws is None else ws.data_ptr(),
                       None, 0, 0, None, None, None, _raw_stream(index))
    st = _lib.lib().wnv_recurrence_forward(index, C.byref(a))
    if st:
        check(st)
    return y, h_last, saved


def _backward(ctx, dy, dh_last):
    z, saved, lengths, seg_start = ctx.saved_tensors
    gates = ctx.gates
    B, T, N = z.shape
    n = N // gates
    code, dev, index = _DTYPES[z.dtype], z.device, z.get_device()
    needs_z, needs_h0 = ctx.needs_input_grad[:2]
    ws_bytes = _sizes(B, T, n, gates, code)[1]
    dz = z.new_empty((B, T, N))
    dh0 = torch.empty((B, n), dtype=torch.float32, device=dev) if needs_h0 else None
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    if dh_last is not None:
        dh_last = dh_last.contiguous()
    zb, zt, _ = z.stride()
    db = dt = 0
    if dy is not None:
        dy = _rows(dy)
        db, dt, _ = dy.stride()
    a = RecurrenceArgs(B, n, T, gates, code, z.data_ptr(), zb, zt, None, 0, None if lengths is None else lengths.data_ptr(),
                       None if seg_start is None else seg_start.data_ptr(), None, None, saved.data_ptr(),
                       None if ws is None else ws.data_ptr(), None if dy is None else dy.data_ptr(), db, dt,
                       None if dh_last is None else dh_last.data_ptr(), dz.data_ptr(), None if dh0 is None else dh0.data_ptr(),
                       _raw_stream(index))
    st = _lib.lib().wnv_recurrence_backward(index, C.byref(a))
    if st:
        check(st)
    return (dz if needs_z else None), dh0, None, None, None


_backward_once = once_differentiable(_backward)


class _GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, h0, gates, lengths, seg_start):
        ctx.set_materialize_grads(False)
        y, h_last, saved = _forward(z, h0, gates, lengths, seg_start, True)
        ctx.gates = gates
        ctx.save_for_backward(z, saved, lengths, seg_start)       # what h0 did is in `saved`: its owner may go on with it
        return y, h_last

    @staticmethod
    def backward(ctx, dy, dh_last):
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, dy, dh_last)


def gated_recurrence(z: torch.Tensor, h0: Optional[torch.Tensor] = None, *, output_gate: bool = True,
                     lengths: Optional[torch.Tensor] = None, seg_start: Optional[torch.Tensor] = None
                     ) -> Tuple[torch.Tensor, torch.Tensor]:
    """z (B, T, 3 C) -> y (B, T, C) of z's type and the state behind the last step (B, C) float32; ``output_gate=False``: z (B, T, 2 C).

    ``h0`` (B, C) float32: the state before the first step (zeros).  ``lengths`` (B,): rows of a padded batch end there -- behind it z
    is not looked at, y and the gradients are zero, and the state is handed on (an empty row's is ``h0``).  ``seg_start`` (B, T): the
    map of a packed slot (``wnv_generate_args``) -- the state reads as zero at each step t with ``seg_start[b, t] == t``; a negative
    entry is an utterance begun before this call, which goes on from ``h0``.  Differentiable (once, not in forward mode) in z and h0.
    Runs on the current stream of z's device and is capturable; the same call gives the same bits, and a row's do not depend on its batch.
    Parts of a long sequence wait for each other on the device; should one not answer for seconds, what depends on it is NaN."""
    if getattr(forward_ad, "_current_level", 0) >= 0:
        refuse_tangents("gated_recurrence", z, h0)
    require_gpu_tensor(z, "z")
    _dtype(z)
    if z.dim() != 3:
        raise ValueError(f"z is {tuple(z.shape)}, expected (B, T, channels)")
    gates = 3 if output_gate else 2
    B, T, n = z.shape
    if B == 0 or T == 0 or n == 0 or n % gates:
        raise ValueError(f"z is {tuple(z.shape)}, expected (B, T, {gates} gates of the same size), none of them empty")
    n //= gates
    z = _rows(z)
    if h0 is not None:
        h0 = _rows(_state(h0, "h0", B, n, z))
    if lengths is not None:
        lengths = _map(lengths, "lengths", (B,), z)
    if seg_start is not None:
        seg_start = _map(seg_start, "seg_start", (B, T), z)
    if torch.is_grad_enabled() and (z.requires_grad or (h0 is not None and h0.requires_grad)):
        return _GatedRecurrence.apply(z, h0, gates, lengths, seg_start)
    y, h_last, _ = _forward(z, h0, gates, lengths, seg_start, False)
    return y, h_last


_step = None


def _load_step():
    global _step
    _step = _lib.lib().wnv_recurrence_step
    return _step


def gated_recurrence_step(z: torch.Tensor, state: torch.Tensor, *, output_gate: bool = True) -> torch.Tensor:
    """One step: z (B, 3 C) (``output_gate=False``: (B, 2 C)), ``state`` (B, C) float32 contiguous, updated in place -> y (B, C) of z's
    type.  Not differentiable: the training form is ``gated_recurrence``."""
    if getattr(forward_ad, "_current_level", 0) >= 0:
        refuse_tangents("gated_recurrence_step", z, state)
    shape, sshape, gates, dev = z.shape, state.shape, 3 if output_gate else 2, z.get_device()
    code = _DTYPES.get(z.dtype)
    if (code is None or dev < 0 or len(shape) != 2 or len(sshape) != 2 or sshape[0] != shape[0] or sshape[1] * gates != shape[1]
            or not z.numel() or state.dtype != torch.float32 or state.get_device() != dev or not state.is_contiguous()
            or ((z.requires_grad or state.requires_grad) and torch.is_grad_enabled())):
        _refuse_step(z, state, gates)
    B, n = sshape
    z = _rows(z)
    y = z.new_empty(sshape)
    increment_version(state)            # a graph that saved the state has to see that it changed
    st = (_step or _load_step())(dev, z.data_ptr(), z.stride(0), state.data_ptr(), y.data_ptr(), B, n, gates, code, _raw_stream(dev))
    if st:
        check(st)
    return y


def _refuse_step(z, state, gates):
    require_gpu_tensor(z, "z")
    _dtype(z)
    if z.dim() != 2 or not z.numel() or z.shape[1] % gates:
        raise ValueError(f"z is {tuple(z.shape)}, expected (B, {gates} gates of the same size), neither of them empty")
    if not _state(state, "state", z.shape[0], z.shape[1] // gates, z).is_contiguous():
        raise ValueError("state is updated in place: it has to be contiguous")
    raise RuntimeError("gated_recurrence_step is not differentiable: use gated_recurrence, or torch.no_grad()")
