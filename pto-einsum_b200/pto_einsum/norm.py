"""Group norm over channels-last tensors, with silu or a silu gate (csrc/pe_norm.cu).

Per row of x [N, ..., C] and group of C / groups channels, over the places of the middle
axes and the group's channels:

    xn = (x - mean) / sqrt(var + eps),   v = xn weight + bias
    out = v  |  silu(v)  |  v silu(gate)

With x [tokens, C] (no middle axes) it is the per-head norm after a recurrent mixer,
and `gate` the mixer's output gate; with x [N, height, width, C] the norm of a feature
map. Differentiable in x, weight, bias and gate; statistics and sums are fp32 and added
in a fixed order.
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import _ops
from ._ops import DTYPES, call, check_tensor, packer, plan, ptr, rows, sig, stride, wants_grad

__all__ = ["group_norm", "group_norm_reference"]

_NORM = packer("6q" "d" "4Q" "4q" "Q" "2Q" "Qq")
_NORM_GRAD = packer("6q" "d" "4Q" "4q" "Q" "2Q" "Qq" "Q" "2q" "4Q" "Qq")


def _fields(lay, x, weight, bias, gate, out, stats):
    """stats [2, N, G]: means, then reciprocal deviations."""
    ints, strides, _ = lay
    mean = ptr(stats)
    return (*ints, x.data_ptr(), ptr(weight), ptr(bias), ptr(gate), *strides, ptr(out), mean,
            mean + 4 * ints[2] * ints[5] if mean else 0)


def _forward(lay, x, weight, bias, gate, stats):
    dev = x.device
    out = _ops.empty(x)
    stats = torch.empty((2, lay[0][2], lay[0][5]), dtype=torch.float32, device=dev) if stats else None
    fields = _fields(lay, x, weight, bias, gate, out, stats)
    nbytes = _ops.nbytes_of("pe_group_norm_ws_bytes", lay, lambda: _NORM.pack(*fields, 0, 0))
    ws = _ops.workspace(nbytes, dev)
    call("pe_group_norm", _NORM.pack(*fields, ptr(ws), nbytes), lay[2])
    return out, stats


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, gate, lay):
        out, stats = _forward(lay, x, weight, bias, gate, True)
        ctx.save_for_backward(x, weight, bias, gate, stats)
        ctx.lay = lay
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        x, weight, bias, gate, stats = ctx.saved_tensors
        lay, dev = ctx.lay, x.device
        dout = _fold(dout)

        dx, dw, db, dgate = [None if t is None else _ops.empty(t) for t in (x, weight, bias, gate)]
        fields = (*_fields(lay, x, weight, bias, gate, None, stats), 0, 0, dout.data_ptr(), *_strides(dout),
                  dx.data_ptr(), ptr(dgate), ptr(dw), ptr(db))
        nbytes = _ops.nbytes_of("pe_group_norm_grad_ws_bytes", lay, lambda: _NORM_GRAD.pack(*fields, 0, 0))
        ws = _ops.workspace(nbytes, dev)
        call("pe_group_norm_grad", _NORM_GRAD.pack(*fields, ptr(ws), nbytes), lay[2])
        return dx, dw, db, dgate, None


def _fold(t):
    """`t` itself, or a copy, such that its middle axes are one axis of one stride."""
    t = rows(t)
    if t.dim() <= 3:
        return t
    try:
        t.view(t.shape[0], -1, t.shape[-1]) if t.numel() else None
        return t
    except RuntimeError:
        return t.contiguous()


def _strides(t):
    """Strides of a row and of a place (0 for an axis of one)."""
    if t.dim() == 2:
        return stride(t, 0), 0
    places = [i for i in range(1, t.dim() - 1) if t.shape[i] > 1]
    return stride(t, 0), stride(t, places[-1]) if places else 0


def group_norm(x, groups: int, weight=None, bias=None, *, eps: float = 1e-5, activation=None, gate=None):
    """Group norm of x [N, ..., C] (channels last) over `groups` groups of channels.

    weight and bias [C] and gate (x's shape) have x's type; activation is None or
    "silu" and excludes a gate. The channels are contiguous; other strides are free
    where the middle axes fold into one. Returns a contiguous tensor of x's shape."""
    try:
        key = ("norm", groups, eps, activation, sig(x), sig(weight), sig(bias), sig(gate))
        lay = plan(key)
    except (AttributeError, TypeError):      # not tensors: the checks say which
        key = lay = None
    if lay is None:
        if activation not in (None, "silu"):
            raise ValueError(f"activation must be None or 'silu' (got {activation!r})")
        if activation and gate is not None:
            raise ValueError("activation and gate exclude each other")
        if not isinstance(x, torch.Tensor) or x.dim() < 2:
            raise ValueError("x must be a tensor of at least two dimensions, channels last")
        _ops.check_activations("x", x, (x.dim(),))
        C = x.shape[-1]
        if groups < 1 or C < 1 or C % groups:
            raise ValueError(f"groups must divide the {C} channels (got {groups})")
        if not eps >= 0:
            raise ValueError(f"eps must not be negative (got {eps})")
        for name, t in (("weight", weight), ("bias", bias)):
            if t is not None:
                check_tensor(name, t, (C,), x.dtype, x.device)
        if gate is not None:
            check_tensor("gate", gate, x.shape, x.dtype, x.device)
        given = (x, weight, bias, gate)
        x, gate = _fold(x), None if gate is None else _fold(gate)
        weight = None if weight is None else weight.contiguous()
        bias = None if bias is None else bias.contiguous()
        places = math.prod(x.shape[1:-1])
        lay = ((DTYPES[x.dtype], 1 if activation else 0, x.shape[0], places, C, int(groups), float(eps)),
               (*_strides(x), *((0, 0) if gate is None else _strides(gate))), x.device.index)
        if key is not None and all(a is b for a, b in zip(given, (x, weight, bias, gate))):
            _ops.keep_plan(key, lay)
    if wants_grad(x, weight, bias, gate):
        return _GroupNorm.apply(x, weight, bias, gate, lay)
    return _forward(lay, x, weight, bias, gate, False)[0]


def group_norm_reference(x, groups, weight=None, bias=None, *, eps=1e-5, activation=None, gate=None):
    """From the definition, in float64 and differentiable, on any device."""
    xg = (x.double().flatten(1, -2) if x.dim() > 2 else x.double().unsqueeze(1)).unflatten(-1, (groups, -1))
    d = xg - xg.mean((1, 3), keepdim=True)
    v = (d / torch.sqrt((d * d).mean((1, 3), keepdim=True) + eps)).reshape(x.shape)
    v = v if weight is None else v * weight.double()
    v = v if bias is None else v + bias.double()
    if activation:
        return v * torch.sigmoid(v)
    return v if gate is None else v * gate.double() * torch.sigmoid(gate.double())
