"""Gated linear recurrence: the PLIF membrane without its spike, the gate of each step taken from a raw
projection.

    f[t] = sigmoid(raw_gate[t] + bias)
    h[t] = f[t] * h[t-1] + (1 - f[t]) * x[t]          y[t] = h[t]

The update is that of ``PLIFNode`` (``v = beta*v + (1-beta)*x``, atomic_ops/plif_node.py:117-134) with a gate
per step. Beside ``parallel_scan.linear_recurrence``, which takes finished coefficients and walks the time
axis of every column in one piece, this one evaluates the gate while it loads, cuts the time axis so that a
few columns fill the GPU too, takes packed sequences of different lengths, and has a form for one token at a
time. The reference has no counterpart.

    gated_linear_recurrence(raw_gate, x, h0=None, bias=None, cu_seqlens=None) -> (y, h_last)
    gated_linear_recurrence_step(raw_gate, x, h, bias=None) -> y        # h updated in place

CUDA tensors only. The state and all sums are fp32 whatever the type of ``x``.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import NSBError
from .parallel_scan import _cast, _common_stream_dtype


def _strided(t: torch.Tensor, dt: torch.dtype):
    """``t`` in the call's element type with unit stride along its last dimension. A view that has that
    already - half of a merged projection, say - is taken as it is."""
    if t.dtype != dt:
        return _lib.convert(t, dt)
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _sizes(t: torch.Tensor):
    """(T, B, D) of a [T, B, D] or [T, D] tensor."""
    return t.shape if t.dim() == 3 else (t.shape[0], 1, t.shape[1])


def _strides(t: torch.Tensor):
    """Strides of T and B in elements."""
    s = t.stride()
    return s[:2] if len(s) == 3 else (s[0], t.shape[1])


def _f32(t, shape, what):
    if t is None:
        return None
    if t.shape != shape:
        raise NSBError(f"{what} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    t = t.detach()
    return t.contiguous() if t.dtype == torch.float32 else t.to(torch.float32).contiguous()


class GatedLinearRecurrence(torch.autograd.Function):
    """``(y, h_last)``; gradients for raw_gate, x, h0 and bias, through both outputs."""

    @staticmethod
    def forward(ctx, raw_gate, x, h0, bias, cu, needs_grad):
        dt = x.dtype if raw_gate.dtype == x.dtype else _common_stream_dtype(raw_gate, x)
        code = _lib.dtype_code(dt)
        a, v = _strided(raw_gate, dt), _strided(x, dt)
        T, B, D = _sizes(x)
        seqs = cu.shape[0] - 1 if cu is not None else 0
        state = torch.Size((seqs, D)) if cu is not None else x.shape[1:]
        h0_32, bias_32 = _f32(h0, state, "h0"), _f32(bias, x.shape[-1:], "bias")
        dev = _lib.require_cuda(a, v, h0_32, bias_32, cu)
        L, at = _lib.lib(), _lib.address
        y = torch.empty(x.shape, dtype=dt, device=dev)
        h_last = torch.empty(state, dtype=torch.float32, device=dev)
        chunks, words = L.nsb_gated_chunks(T), L.nsb_gated_scratch_words(T, B * D)
        ckpt = torch.empty(chunks * B * D, dtype=torch.float32, device=dev) if needs_grad and chunks > 1 else None
        scratch = torch.empty(words, dtype=torch.int32, device=dev) if words else None
        _lib.launch(dev, "nsb_gated_recurrence_fwd", at(a), *_strides(a), at(v), *_strides(v), at(bias_32), at(h0_32),
                    at(cu), seqs, at(y), at(h_last), at(ckpt), at(scratch), T, B, D, code)
        if needs_grad:
            ctx.save_for_backward(a, v, h0_32, bias_32, cu, ckpt)
            ctx.in_dtypes = (raw_gate.dtype, x.dtype, h0.dtype if h0 is not None else None,
                             bias.dtype if bias is not None else None)
            ctx.state = state
            ctx.set_materialize_grads(False)
        return (y if dt == x.dtype else _cast(y, x.dtype)), h_last

    @staticmethod
    def backward(ctx, dy, dh_last):
        if torch.is_grad_enabled():  # (create_graph=True)
            raise NSBError("gated_linear_recurrence has no second derivatives")
        a, v, h0, bias, cu, ckpt = ctx.saved_tensors
        T, B, D = _sizes(v)
        dev, dt, L, at = a.device, a.dtype, _lib.lib(), _lib.address
        dy = torch.zeros(v.shape, dtype=dt, device=dev) if dy is None else _lib.convert(dy, dt)
        dh = None if dh_last is None else dh_last.contiguous()
        want_a, want_x, want_h, want_b = ctx.needs_input_grad[:4]
        d_raw = torch.empty(a.shape, dtype=dt, device=dev) if want_a else None
        d_x = torch.empty(v.shape, dtype=dt, device=dev) if want_x else None
        d_h0 = torch.empty(ctx.state, dtype=torch.float32, device=dev) if want_h and h0 is not None else None
        d_bias = torch.empty(D, dtype=torch.float32, device=dev) if want_b and bias is not None else None
        words = L.nsb_gated_scratch_words(T, B * D)  # (a multiple of 16 bytes)
        sums = L.nsb_gated_chunks(T) * B * D if d_bias is not None else 0
        scratch = torch.empty(words + sums, dtype=torch.float32, device=dev) if words + sums else None
        part = scratch.data_ptr() + 4 * words if sums else None
        _lib.launch(dev, "nsb_gated_recurrence_bwd", at(a), *_strides(a), at(v), *_strides(v), at(bias), at(h0), at(cu),
                    cu.shape[0] - 1 if cu is not None else 0, at(ckpt), at(dy), at(dh), at(d_raw), at(d_x), at(d_bias),
                    at(d_h0), part, at(scratch), T, B, D, _lib.dtype_code(dt))
        return (*(g if g is None or g.dtype == t else _cast(g, t) for g, t in zip((d_raw, d_x, d_h0, d_bias), ctx.in_dtypes)),
                None, None)


def gated_linear_recurrence(raw_gate: torch.Tensor, x: torch.Tensor, h0: torch.Tensor | None = None,
                            bias: torch.Tensor | None = None, cu_seqlens: torch.Tensor | None = None):
    """``raw_gate``, ``x``: [T, B, D], time-major as in the scans of ``parallel_scan``, or [T, D]. They may be
    views with unit stride along D (halves of one projection); differing types are widened to fp32. ``h0``:
    state before the first step, [B, D] (or [D]), zeros if None. ``bias``: [D], added to ``raw_gate``. Returns
    ``y`` in ``x``'s shape and type and ``h_last``, the fp32 state after the last step.

    Packed sequences: ``raw_gate`` and ``x`` [rows, D] and ``cu_seqlens``, seqs + 1 integers on the device that do
    not decrease; sequence s is rows ``cu_seqlens[s]`` to ``cu_seqlens[s+1] - 1`` and has ``h0[s]`` and
    ``h_last[s]`` ([seqs, D]). A sequence may be empty; rows outside of all sequences get zero, in ``y`` and in
    the gradients. Nothing, NaN included, passes from one sequence to another. The values of ``cu_seqlens`` are not looked at
    by the host; they have to lie in 0 .. rows (a sequence whose last row is not there leaves its ``h_last`` unwritten).

    An infinite state goes on as infinite or NaN. There are no second derivatives: a backward pass with
    ``create_graph=True`` is refused.

    Inputs must not be changed in place between forward and backward. The first call of a process must not be
    made inside a CUDA stream capture (nor may that of the scans; it sets up the library's error word)."""
    if raw_gate.shape != x.shape or x.dim() not in (2, 3):
        raise NSBError(f"gated_linear_recurrence expects raw_gate and x of one shape [T, B, D] or [T, D], got "
                       f"{tuple(raw_gate.shape)} and {tuple(x.shape)}")
    if cu_seqlens is not None:
        if x.dim() != 2 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
            raise NSBError("packed sequences: raw_gate and x are [rows, D], cu_seqlens has seqs + 1 elements")
        if cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise NSBError(f"cu_seqlens has type {cu_seqlens.dtype}; expected int32 or int64")
        cu_seqlens = cu_seqlens.to(torch.int32).contiguous()
    return GatedLinearRecurrence.apply(raw_gate, x, h0, bias, cu_seqlens, _lib.wants_gradients(raw_gate, x, h0, bias))


def gated_linear_recurrence_step(raw_gate: torch.Tensor, x: torch.Tensor, h: torch.Tensor,
                                 bias: torch.Tensor | None = None) -> torch.Tensor:
    """One token for each of B running sequences: ``raw_gate``, ``x`` [B, D]; the fp32 state ``h`` [B, D] is
    updated in place and returned rounded to ``x``'s type. No gradients; to autograd it is a change in place of ``h``."""
    if x.dim() != 2 or raw_gate.shape != x.shape or h.shape != x.shape:
        raise NSBError("gated_linear_recurrence_step expects raw_gate, x and h of one shape [B, D]")
    if h.dtype != torch.float32 or not h.is_contiguous():
        raise NSBError("gated_linear_recurrence_step: h must be a contiguous float32 tensor (it is updated in place)")
    if torch.is_grad_enabled() and (raw_gate.requires_grad or x.requires_grad or h.requires_grad
                                    or (bias is not None and bias.requires_grad)):
        raise NSBError("gated_linear_recurrence_step has no gradients; use gated_linear_recurrence, or torch.no_grad()")
    dt = x.dtype if raw_gate.dtype == x.dtype else _common_stream_dtype(raw_gate, x)
    code = _lib.dtype_code(dt)
    a, v, b = _strided(raw_gate, dt), _strided(x, dt), _f32(bias, x.shape[1:], "bias")
    dev = _lib.require_cuda(a, v, h, b)
    y = torch.empty(x.shape, dtype=dt, device=dev)
    at = _lib.address
    _lib.launch(dev, "nsb_gated_recurrence_step", at(a), a.stride(0), at(v), v.stride(0), at(b), at(h), at(y), x.shape[0],
                x.shape[1], code)
    if not h.is_inference():  # a graph that has saved h must not take the new state for the old one
        torch.autograd.graph.increment_version(h)
    return y if dt == x.dtype else _cast(y, x.dtype)
