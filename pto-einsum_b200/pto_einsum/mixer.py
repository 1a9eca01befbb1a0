"""A selective state space mixer layer: contractions, convolution, scan and norm together.

    x, z    = split(h w_in)                        'bte,ef->btf'
    x       = silu(causal_conv(x))
    r, B, C = split(x w_x)                         'btd,dr->btr'
    delta   = r w_dt                               'btr,rd->btd'
    y       = selective_scan(x, delta, A, B, C, D)
    out     = (group_norm(y) silu(z)) w_out        'btd,de->bte'

The projections are two-operand contractions of this library, one cached runner per
(equation, shapes, dtype) as in `pto_einsum.gdn`; the rest are `pto_einsum.ssm` and
`pto_einsum.norm`. `forward` takes prompts (a batch or packed sequences) and returns the
layer's state; `step` takes one token of each request and updates that state in place.
Gradients flow through every operator, the contractions included (their gradients are
contractions of the same labels), so a training step is forward, backward, update.

Example:
    >>> mix = SelectiveMixer(width=256, channels=512, states=16, heads=8, device="cuda")
    >>> y, state = mix(prompt, return_state=True)   # prompt [B, T, 256]
    >>> y1 = mix.step(token, state)                 # token [B, 256]
"""
from __future__ import annotations

import math

import torch

from .gdn import GDNChunked
from .norm import group_norm
from .ssm import causal_conv, causal_conv_step, selective_scan, selective_scan_step

__all__ = ["SelectiveMixer", "contract"]


class _Contract(torch.autograd.Function):
    """out = einsum('X,Y->Z'); dX = einsum('Z,Y->X'), dY = einsum('X,Z->Y')."""

    @staticmethod
    def forward(ctx, backend, eq, a, b):
        ctx.save_for_backward(a, b)
        ctx.plan = backend, eq
        return backend.contract(eq, a, b).to(a.dtype)

    @staticmethod
    def backward(ctx, dout):
        a, b = ctx.saved_tensors
        backend, eq = ctx.plan
        ins, z = eq.replace(" ", "").split("->")
        x, y = ins.split(",")
        # by the differentiable form: gradients of gradients are contractions again
        da = contract(backend, f"{z},{y}->{x}", dout, b).to(a.dtype) if ctx.needs_input_grad[2] else None
        db = contract(backend, f"{x},{z}->{y}", a, dout).to(b.dtype) if ctx.needs_input_grad[3] else None
        return None, None, da, db


def contract(backend: GDNChunked, eq: str, a, b):
    """A contraction on the backend's runners, in the operands' type, differentiable any
    number of times. Every label of an operand has to appear in the other operand or the
    output."""
    return _Contract.apply(backend, eq, a, b)


class SelectiveMixer:
    """width: of the layer's input and output; channels: of the scan; states: per channel;
    heads: groups of the norm; groups: of B and C; rank: of the step size (width / 16
    rounded up by default); taps: of the convolution. dtype float16 or float32 (the types
    of the contractions). Parameters are plain tensors in `params`, seeded."""

    def __init__(self, width: int, channels: int, states: int = 16, heads: int = 1, groups: int = 1, rank=None,
                 taps: int = 4, dtype: torch.dtype = torch.float16, device="cuda", seed: int = 0,
                 requires_grad: bool = False):
        if dtype not in (torch.float16, torch.float32):
            raise TypeError(f"dtype must be float16 or float32 (got {dtype})")
        if channels % heads or channels % groups:
            raise ValueError("heads and groups must divide the channels")
        self.channels, self.states, self.heads, self.groups = channels, states, heads, groups
        self.rank = rank if rank else -(-width // 16)
        self.taps, self.dtype = taps, dtype
        self.backend = GDNChunked("pto", dtype=dtype)
        gen = torch.Generator().manual_seed(seed)

        def normal(*shape, fan):
            return (torch.randn(shape, generator=gen) * fan ** -0.5).to(device=device, dtype=dtype)

        cols = self.rank + 2 * groups * states
        step = torch.exp(torch.rand(channels, generator=gen) * math.log(100.0)) * 1e-3   # 0.001 to 0.1
        f32 = dict(device=device, dtype=torch.float32)
        self.params = {
            "w_in": normal(width, 2 * channels, fan=width), "w_x": normal(channels, cols, fan=channels),
            "w_dt": normal(self.rank, channels, fan=self.rank), "w_out": normal(channels, width, fan=channels),
            "conv_w": normal(channels, taps, fan=taps), "conv_b": normal(channels, fan=100.0),
            "A_log": torch.arange(1, states + 1).float().log().expand(channels, states).contiguous().to(**f32),
            "D": torch.ones(channels, **f32), "dt_bias": (step + torch.log(-torch.expm1(-step))).to(**f32),
            "norm_w": torch.ones(channels, device=device, dtype=dtype),
            "norm_b": torch.zeros(channels, device=device, dtype=dtype)}
        for p in self.params.values():
            p.requires_grad_(requires_grad)

    def empty_state(self, slots: int):
        """State of `slots` requests before their first token, for `step`."""
        dev = self.params["D"].device
        return {"conv": torch.zeros(slots, self.taps - 1, self.channels, dtype=self.dtype, device=dev),
                "ssm": torch.zeros(slots, self.channels, self.states, device=dev)}

    def _split(self, cols):
        """r, B, C of the projection's columns (views of it)."""
        gn = self.groups * self.states
        r, b, c = cols.split([self.rank, gn, gn], dim=-1)
        shape = (*cols.shape[:-1], self.groups, self.states)
        return r, b.unflatten(-1, shape[-2:]), c.unflatten(-1, shape[-2:])

    def forward(self, h, state=None, cu_seqlens=None, return_state: bool = False):
        """h [B, T, width] (packed with cu_seqlens) -> [B, T, width], and with return_state the
        state after each sequence."""
        p, Dc = self.params, self.channels
        xz = contract(self.backend, "bte,ef->btf", h, p["w_in"])
        x, z = xz[..., :Dc], xz[..., Dc:]
        x = causal_conv(x, p["conv_w"], p["conv_b"], activation="silu", cu_seqlens=cu_seqlens,
                        initial_state=state["conv"] if state else None, return_state=return_state)
        x, conv = x if return_state else (x, None)
        r, B, C = self._split(contract(self.backend, "btd,dr->btr", x, p["w_x"]))
        delta = contract(self.backend, "btr,rd->btd", r, p["w_dt"])
        y = selective_scan(x, delta, -torch.exp(p["A_log"]), B, C, p["D"], delta_bias=p["dt_bias"],
                           delta_softplus=True, cu_seqlens=cu_seqlens, initial_state=state["ssm"] if state else None,
                           return_state=return_state)
        y, ssm = y if return_state else (y, None)
        y = group_norm(y.flatten(0, 1), self.heads, p["norm_w"], p["norm_b"], gate=z.flatten(0, 1))
        out = contract(self.backend, "btd,de->bte", y.view(x.shape), p["w_out"])
        return (out, {"conv": conv, "ssm": ssm}) if return_state else out

    __call__ = forward

    def step(self, h, state, slots=None):
        """One token h [B, width] of each request; `state` is updated in place (row slots[b]
        of it, row b without slots)."""
        p, Dc = self.params, self.channels
        with torch.no_grad():
            xz = contract(self.backend, "be,ef->bf", h, p["w_in"])
            x, z = xz[:, :Dc], xz[:, Dc:]
            x = causal_conv_step(x, state["conv"], p["conv_w"], p["conv_b"], activation="silu", slots=slots)
            r, B, C = self._split(contract(self.backend, "bd,dr->br", x, p["w_x"]))
            delta = contract(self.backend, "br,rd->bd", r, p["w_dt"])
            y = selective_scan_step(state["ssm"], x, delta, -torch.exp(p["A_log"]), B, C, p["D"],
                                    delta_bias=p["dt_bias"], delta_softplus=True, slots=slots)
            y = group_norm(y, self.heads, p["norm_w"], p["norm_b"], gate=z)
            return contract(self.backend, "bd,de->be", y, p["w_out"])

    def cleanup(self):
        self.backend.cleanup()
