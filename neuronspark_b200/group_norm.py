"""Group norm with an activation, channels last.

    xh = (x - mean) / sqrt(var + eps)      z = weight * xh + bias      y = z * sigmoid(z)   (or y = z)

The statistics of a sample and a group of C / num_groups channels go over all positions of the sample: ``x`` is
[N, ..., C]. An [N, C] tensor has one position per sample, so every row's groups are normalised by themselves:
what the heads of a recurrence's output want, token by token (reshape a time-major [T, B, D] to [T*B, D]).

Beside ``lateral_inhibition.LateralInhibition`` / ``RMSNorm``, which normalise whole rows by their mean square;
the reference has no group norm. CUDA tensors only; statistics and sums are fp32 whatever the type of ``x``.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib
from ._lib import NSBError

_ACTIVATIONS = {None: _lib.ACT_NONE, "silu": _lib.ACT_SILU}


def _param(t):
    if t is None:
        return None
    t = t.detach()
    return t.contiguous() if t.dtype == torch.float32 else t.to(torch.float32).contiguous()


class GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, num_groups, eps, act, needs_grad):
        x_c, w, b = x.contiguous(), _param(weight), _param(bias)
        dev = _lib.require_cuda(x_c, w, b)
        shape = x.shape
        N, C = shape[0], shape[-1]
        L = x_c.numel() // (N * C) if N * C else 0
        lib, at = _lib.lib(), _lib.address
        y = torch.empty(shape, dtype=x.dtype, device=dev)
        stats = torch.empty(2 * N * num_groups, dtype=torch.float32, device=dev) if needs_grad else None
        words = lib.nsb_group_norm_scratch_floats(N, L, C, num_groups, 0)
        scratch = torch.empty(words, dtype=torch.float32, device=dev) if words else None
        mean = at(stats)
        rstd = mean + 4 * N * num_groups if mean else None
        _lib.launch(dev, "nsb_group_norm_fwd", at(x_c), at(w), at(b), at(y), mean, rstd, at(scratch), N, L, C, num_groups,
                    eps, act, _lib.dtype_code(x.dtype))
        if needs_grad:
            ctx.save_for_backward(x_c, w, b, stats)
            ctx.sizes = (N, L, C, num_groups, act)
            ctx.in_dtypes = (weight.dtype if weight is not None else None, bias.dtype if bias is not None else None)
        return y

    @staticmethod
    def backward(ctx, grad_out):
        if torch.is_grad_enabled():  # (create_graph=True)
            raise NSBError("group_norm_act has no second derivatives")
        x, w, b, stats = ctx.saved_tensors
        N, L, C, G, act = ctx.sizes
        dev, lib, at = x.device, _lib.lib(), _lib.address
        dy = _lib.convert(grad_out, x.dtype)
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
        dw = torch.empty(C, dtype=torch.float32, device=dev) if need_w and w is not None else None
        db = torch.empty(C, dtype=torch.float32, device=dev) if need_b and b is not None else None
        words = lib.nsb_group_norm_scratch_floats(N, L, C, G, 1)
        scratch = torch.empty(words, dtype=torch.float32, device=dev) if words else None
        mean = at(stats)
        rstd = mean + 4 * N * G if mean else None
        _lib.launch(dev, "nsb_group_norm_bwd", at(dy), at(x), at(w), at(b), mean, rstd, at(dx), at(dw), at(db), at(scratch),
                    N, L, C, G, act, _lib.dtype_code(x.dtype))
        return (dx, *(g if g is None or g.dtype == t else g.to(t) for g, t in zip((dw, db), ctx.in_dtypes)), None, None, None,
                None)


def group_norm_act(x: torch.Tensor, num_groups: int, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                   eps: float = 1e-5, activation: str | None = "silu") -> torch.Tensor:
    """``x`` [N, ..., C] (float32, bfloat16 or float16), ``weight`` and ``bias`` [C] or None. ``activation`` is
    "silu" or None. Returns a contiguous tensor of ``x``'s shape and type; gradients for x, weight and bias. There are no
    second derivatives: a backward pass with ``create_graph=True`` is refused.

    Made for groups of up to 256 channels where a sample has one position, and for samples of 64 positions and more
    otherwise. Wider groups and shorter samples are right but slow (65536 x 768 in 2 groups takes longer than elementary torch
    operations), and their backward pass takes 8 bytes of workspace per sample and channel."""
    if x.dim() < 2:
        raise NSBError("group_norm_act expects x of [N, ..., C]")
    C = x.shape[-1]
    if num_groups < 1 or C % num_groups:
        raise NSBError(f"group_norm_act: {C} channels do not divide into {num_groups} groups")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) != (C,):
            raise NSBError(f"{name} has shape {tuple(t.shape)}, expected {(C,)}")
    if activation not in _ACTIVATIONS:
        raise NSBError(f"unknown activation {activation!r}; expected 'silu' or None")
    _lib.dtype_code(x.dtype)
    return GroupNormAct.apply(x, weight, bias, int(num_groups), float(eps), _ACTIVATIONS[activation],
                              _lib.wants_gradients(x, weight, bias))


class GroupNorm(nn.Module):
    """``group_norm_act`` with its parameters, channels last."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, activation: str | None = "silu"):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(num_channels))
        self.bias = nn.Parameter(torch.zeros(num_channels))
        self.num_groups, self.eps, self.activation = num_groups, eps, activation

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return group_norm_act(x, self.num_groups, self.weight, self.bias, self.eps, self.activation)

    def extra_repr(self):
        return f"{self.num_groups}, {self.weight.numel()}, eps={self.eps}, activation={self.activation}"
