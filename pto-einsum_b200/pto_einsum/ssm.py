"""Short causal convolution and selective state space scan, for prompts and single tokens.

The operators of a recurrent mixer layer that are not contractions, as hand-written
sm_100a kernels (csrc/pe_conv.cu, csrc/pe_scan.cu). Activations are channels last,
[batch, token, channel], float32, float16 or bfloat16; states and sums are fp32.

Causal convolution, one filter of W = 2 to 4 taps a channel:

    p[t] = bias + sum_k weight[c, k] x[t - (W - 1) + k],   out = p  or  silu(p)

Selective scan (Gu and Dao, "Mamba: Linear-Time Sequence Modeling with Selective State
Spaces", 2023, algorithm 2), per channel d of group g and state n:

    dt = delta + delta_bias,  through softplus if asked
    h[n] = exp(dt A[d, n]) h[n] + dt u B[g, n]
    out = (sum_n C[g, n] h[n] + D[d] u) silu(z)

Packed prompts: with ``cu_seqlens`` (S + 1 rising offsets, as in `pto_einsum.gdn`, but
any lengths, empty ones too) the batch is one row that holds S sequences. A list or a
host tensor is checked by the host and copied, which waits for the stream; an int32
tensor on the device costs no synchronisation, and a wrong one shows in
`_core.device_error`.

Both prompt operators are differentiable in every floating argument. Their gradients
are written by kernels that add in a fixed order: the same inputs give the same bits.
The `_step` forms take one token of each request and update the states in place, in
rows picked by ``slots`` where the states live in a pool (a negative slot skips the
request). A scan step takes up to 65535 requests.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _ops
from ._ops import (DTYPES, call, check_activations, check_tensor, offsets, packer, plan, ptr, rows, sig, stride,
                   wants_grad)

__all__ = ["causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step",
           "causal_conv_reference", "selective_scan_reference", "MAX_STATES"]

MAX_STATES = 128

_CONV = packer("7q" "Q" "4Q" "2q" "2Q")
_CONV_GRAD = packer("7q" "Q" "4Q" "2q" "2Q" "2Q" "2q" "4Q" "Qq")
_CONV_STEP = packer("6q" "2Q" "3Q" "q" "2Q")
_SCAN = packer("8q" "Q" "5Q" "4Q" "12q" "4Q" "q")
_SCAN_GRAD = packer("8q" "Q" "5Q" "4Q" "12q" "4Q" "q" "Q" "2q" "Q" "5Q" "4Q" "Qq")
_SCAN_STEP = packer("7q" "2Q" "5Q" "3Q" "7q" "2Q")


def _silu(activation) -> int:
    if activation not in (None, "silu"):
        raise ValueError(f"activation must be None or 'silu' (got {activation!r})")
    return 1 if activation else 0


# ---- causal convolution -------------------------------------------------------------
def _check_filter(x, weight, bias):
    C = x.shape[-1]
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or not 2 <= weight.shape[1] <= 4:
        raise ValueError(f"weight must be [channels, width] with a width of 2 to 4 "
                         f"(got {tuple(getattr(weight, 'shape', ()))})")
    check_tensor("weight", weight, (C, weight.shape[1]), x.dtype, x.device)
    if bias is not None:
        check_tensor("bias", bias, (C,), x.dtype, x.device)
    if C < 1:
        raise ValueError("x has no channels")
    return weight.shape[1]


def _conv_layout(x, weight, nseq, silu):
    """The numbers of a call, its strides and its device: all but the pointers."""
    return (DTYPES[x.dtype], silu, weight.shape[1], *x.shape, nseq), (stride(x, 0), stride(x, 1)), x.device.index


def _conv_fields(lay, x, weight, bias, init, cu, out, state):
    return (*lay[0], ptr(cu), x.data_ptr(), weight.data_ptr(), ptr(bias), ptr(init), *lay[1], ptr(out), ptr(state))


def _conv_forward(lay, x, weight, bias, init, cu, want_state):
    out = _ops.empty(x)
    state = None
    if want_state:
        _, _, W, _, _, C, nseq = lay[0]
        state = torch.empty((nseq, W - 1, C), dtype=x.dtype, device=x.device)
    call("pe_causal_conv", _CONV.pack(*_conv_fields(lay, x, weight, bias, init, cu, out, state)), lay[2])
    return out, state


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, init, cu, lay, want_state):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, init, cu)
        ctx.lay = lay
        out, state = _conv_forward(lay, x, weight, bias, init, cu, want_state)
        return (out, state) if want_state else out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dstate=None):
        x, weight, bias, init, cu = ctx.saved_tensors
        lay, dev, dt = ctx.lay, x.device, x.dtype
        dout = torch.zeros(x.shape, dtype=dt, device=dev) if dout is None else rows(dout)
        dstate = None if dstate is None else dstate.contiguous()
        dx, dw, db, dinit = _ops.empty(x), _ops.empty(weight), _opt(bias, _ops.empty), _opt(init, _ops.empty)
        fields = (*_conv_fields(lay, x, weight, bias, init, cu, None, None), dout.data_ptr(), ptr(dstate),
                  stride(dout, 0), stride(dout, 1), dx.data_ptr(), ptr(dinit), dw.data_ptr(), ptr(db))
        nbytes = _ops.nbytes_of("pe_causal_conv_grad_ws_bytes", lay, lambda: _CONV_GRAD.pack(*fields, 0, 0))
        ws = _ops.workspace(nbytes, dev)
        call("pe_causal_conv_grad", _CONV_GRAD.pack(*fields, ptr(ws), nbytes), lay[2])
        return dx, dw, db, dinit, None, None, None


def causal_conv(x, weight, bias=None, *, activation=None, initial_state=None, cu_seqlens=None,
                return_state: bool = False):
    """Causal convolution of x [B, T, C] with weight [C, W] (and bias [C]) along the tokens.

    activation: None or "silu". initial_state [S, W - 1, C]: the inputs before each
    sequence (zeros without it). Returns out [B, T, C], and with return_state the last
    W - 1 inputs of each sequence [S, W - 1, C], for `causal_conv_step` or the next
    piece of the prompt. All tensors have x's type; x's channels are contiguous, its
    other strides are free."""
    cu = cu_seqlens
    try:
        key = ("conv", activation, sig(x), sig(weight), sig(bias), sig(initial_state), sig(cu))
        lay = plan(key)
    except (AttributeError, TypeError):      # not tensors: the checks say which
        key = lay = None
    if lay is None:
        silu = _silu(activation)
        check_activations("x", x, (3,))
        W = _check_filter(x, weight, bias)
        B, T, C = x.shape
        cu, nseq = offsets(cu_seqlens, B, T, x.device)
        if initial_state is not None:
            check_tensor("initial_state", initial_state, (nseq, W - 1, C), x.dtype, x.device)
        given = (x, weight, bias, initial_state, cu_seqlens)
        x, weight = rows(x), weight.contiguous()
        bias, initial_state = _opt(bias, torch.Tensor.contiguous), _opt(initial_state, torch.Tensor.contiguous)
        lay = _conv_layout(x, weight, nseq, silu)
        if key is not None and all(a is b for a, b in zip(given, (x, weight, bias, initial_state, cu))):
            _ops.keep_plan(key, lay)
    if wants_grad(x, weight, bias, initial_state):
        return _CausalConv.apply(x, weight, bias, initial_state, cu, lay, return_state)
    out, state = _conv_forward(lay, x, weight, bias, initial_state, cu, return_state)
    return (out, state) if return_state else out


def causal_conv_step(x, state, weight, bias=None, *, activation=None, slots=None):
    """One token x [B, C] of each request; returns out [B, C].

    state [S, W - 1, C] (contiguous, x's type) is shifted in place: row slots[b] of it
    belongs to request b (row b without slots, S = B). Rows with a negative slot give 0
    and touch no state; two requests must not share a slot. There is no gradient: inputs
    that require one are refused outside torch.no_grad()."""
    try:
        key = ("conv step", activation, _ops.sigs(x, state, weight, bias, slots))
        ints = plan(key)
    except (AttributeError, TypeError):      # not tensors: the checks say which
        key = ints = None
    if ints is None:
        silu = _silu(activation)
        check_activations("x", x, (2,))
        W = _check_filter(x, weight, bias)
        B, C = x.shape
        _check_state("state", state, x.dtype, x.device, (W - 1, C), B, slots)
        _ops.check_slots(slots, B, x.device)
        if any(t is not None and not t.is_contiguous() for t in (weight, bias)) or rows(x) is not x:
            key = None
            x, weight = rows(x), weight.contiguous()
            bias = None if bias is None else bias.contiguous()
        ints = (DTYPES[x.dtype], silu, W, B, C, state.shape[0], stride(x, 0), x.device.index,
                _ask_for_gradients(x, state, weight, bias), x.is_contiguous())
        if key is not None:
            _ops.keep_plan(key, ints)
    if ints[8] or forward_ad._current_level >= 0:
        _no_gradients("causal_conv_step", state, x, weight, bias)
    out = torch.empty_like(x) if ints[9] else _ops.empty(x)
    s32, s64 = (0, 0) if slots is None else _ops.slot_pointers(slots)
    call("pe_causal_conv_step", _CONV_STEP.pack(
        *ints[:6], s32, s64, x.data_ptr(), weight.data_ptr(), 0 if bias is None else bias.data_ptr(), ints[6],
        state.data_ptr(), out.data_ptr()), ints[7])
    increment_version(state)   # autograd sees the kernel's writes as its own in-place operations
    return out


def _ask_for_gradients(*tensors) -> bool:
    return any(t is not None and t.requires_grad for t in tensors)


def _no_gradients(name, state, *inputs):
    if state.requires_grad and torch.is_grad_enabled():
        raise ValueError("state is updated in place and cannot require a gradient")
    if wants_grad(state, *inputs):
        raise ValueError(f"{name} has no gradient: call it under torch.no_grad(), or the prompt form on one token")


def _check_state(name, state, dtype, dev, tail, batch, slots):
    if not isinstance(state, torch.Tensor) or state.dim() != 3:
        raise ValueError(f"{name} must have three dimensions, one row of {tail} a slot")
    n = state.shape[0] if slots is not None else batch
    check_tensor(name, state, (n, *tail), dtype, dev)
    if not state.is_contiguous():
        raise ValueError(f"{name} must be contiguous (it is updated in place)")


# ---- selective scan -------------------------------------------------------------------
def _check_scan(u, delta, A, B, C, D, z, delta_bias, lead):
    """Types and shapes; returns B and C as [*lead, G, N]."""
    dt, dev, Dc = u.dtype, u.device, u.shape[-1]
    if Dc < 1:
        raise ValueError("u has no channels")
    if not isinstance(A, torch.Tensor) or A.dim() != 2 or not 1 <= A.shape[1] <= MAX_STATES:
        raise ValueError(f"A must be [channels, states] with 1 to {MAX_STATES} states "
                         f"(got {tuple(getattr(A, 'shape', ()))})")
    N = A.shape[1]
    check_tensor("A", A, (Dc, N), torch.float32, dev)
    for name, t in (("D", D), ("delta_bias", delta_bias)):
        if t is not None:
            check_tensor(name, t, (Dc,), torch.float32, dev)
    check_tensor("delta", delta, u.shape, dt, dev)
    if z is not None:
        check_tensor("z", z, u.shape, dt, dev)
    if not isinstance(B, torch.Tensor) or not isinstance(C, torch.Tensor):
        raise TypeError("B and C must be torch.Tensors")
    if B.dim() == len(lead) + 1:
        B = B.unsqueeze(-2)
    if C.dim() == len(lead) + 1:
        C = C.unsqueeze(-2)
    if B.dim() != len(lead) + 2 or B.shape[-2] < 1 or Dc % B.shape[-2]:
        raise ValueError(f"B must be [..., groups, states] with groups dividing the {Dc} channels "
                         f"(got {tuple(B.shape)})")
    shape = (*lead, B.shape[-2], N)
    check_tensor("B", B, shape, dt, dev)
    check_tensor("C", C, shape, dt, dev)
    return B, C


def _opt(t, f):
    return None if t is None else f(t)


def _scan_layout(u, delta, A, B, C, z, nseq, softplus):
    zs = (0, 0) if z is None else (stride(z, 0), stride(z, 1))
    return ((DTYPES[u.dtype], softplus, *u.shape, A.shape[1], B.shape[-2], nseq),
            (stride(u, 0), stride(u, 1), stride(delta, 0), stride(delta, 1), *zs, stride(B, 0), stride(B, 1),
             stride(B, -2), stride(C, 0), stride(C, 1), stride(C, -2)), u.device.index)


def _scan_fields(lay, u, delta, A, B, C, D, z, bias, h0, cu, out, state, ckpt):
    return (*lay[0], ptr(cu), u.data_ptr(), delta.data_ptr(), ptr(z), B.data_ptr(), C.data_ptr(), A.data_ptr(),
            ptr(D), ptr(bias), ptr(h0), *lay[1], ptr(out), ptr(state), ptr(ckpt))


def _scan_forward(lay, u, delta, A, B, C, D, z, bias, h0, cu, want_state, want_ckpt):
    dev, f32 = u.device, torch.float32
    _, _, _, T, Dc, N, _, nseq = lay[0]
    out = _ops.empty(u)
    state = torch.empty((nseq, Dc, N), dtype=f32, device=dev) if want_state else None
    ckpt = torch.empty(_core_ckpt(T, nseq, cu is not None, Dc, N), dtype=f32, device=dev) if want_ckpt else None
    fields = _scan_fields(lay, u, delta, A, B, C, D, z, bias, h0, cu, out, state, ckpt)
    nbytes = _ops.nbytes_of("pe_scan_ws_bytes", (lay[0] + (cu is None,), 0, lay[2]),
                            lambda: _SCAN.pack(*fields, 0, 0))
    ws = _ops.workspace(nbytes, dev)
    call("pe_selective_scan", _SCAN.pack(*fields, ptr(ws), nbytes), lay[2])
    return out, state, ckpt


def _core_ckpt(tokens, nseq, packed, channels, states) -> int:
    fn = _ops.function("pe_scan_ckpt_floats", restype=ctypes.c_int64, argtypes=[ctypes.c_int64] * 5)
    return fn(tokens, nseq, int(packed), channels, states)


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, bias, h0, cu, lay, want_state):
        ctx.set_materialize_grads(False)
        out, state, ckpt = _scan_forward(lay, u, delta, A, B, C, D, z, bias, h0, cu, want_state, True)
        # not h0: its values are in the checkpoints, and a decode step may go on in its place
        ctx.save_for_backward(u, delta, A, B, C, D, z, bias, cu, ckpt)
        ctx.lay, ctx.has_h0 = lay, h0 is not None
        return (out, state) if want_state else out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dstate=None):
        u, delta, A, B, C, D, z, bias, cu, ckpt = ctx.saved_tensors
        lay, dev, dt = ctx.lay, u.device, u.dtype
        dout = torch.zeros(u.shape, dtype=dt, device=dev) if dout is None else rows(dout)
        dstate = _opt(dstate, torch.Tensor.contiguous)

        du, ddelta, dz, dB, dC, dA, dD, dbias = [_opt(t, _ops.empty) for t in (u, delta, z, B, C, A, D, bias)]
        dh0 = torch.empty((lay[0][7], *A.shape), dtype=torch.float32, device=dev) if ctx.has_h0 else None
        fields = (*_scan_fields(lay, u, delta, A, B, C, D, z, bias, None, cu, None, None, ckpt), 0, 0,
                  dout.data_ptr(), stride(dout, 0), stride(dout, 1), ptr(dstate), ptr(du), ptr(ddelta), ptr(dz),
                  ptr(dB), ptr(dC), ptr(dA), ptr(dD), ptr(dbias), ptr(dh0))
        nbytes = _ops.nbytes_of("pe_scan_grad_ws_bytes", (lay[0] + (cu is None,), 0, lay[2]),
                                lambda: _SCAN_GRAD.pack(*fields, 0, 0))
        ws = _ops.workspace(nbytes, dev)
        call("pe_selective_scan_grad", _SCAN_GRAD.pack(*fields, ptr(ws), nbytes), lay[2])
        return du, ddelta, dA, dB, dC, dD, dz, dbias, dh0, None, None, None


def selective_scan(u, delta, A, B, C, D=None, *, z=None, delta_bias=None, delta_softplus: bool = False,
                   initial_state=None, cu_seqlens=None, return_state: bool = False):
    """Selective scan of u [Bt, T, Dc] with step sizes delta [Bt, T, Dc].

    A [Dc, N], D [Dc] and delta_bias [Dc] are float32; B and C [Bt, T, G, N] (or
    [Bt, T, N], one group) and the gate z [Bt, T, Dc] have u's type, N up to 128,
    channels in G equal groups. initial_state [S, Dc, N] float32 (zeros without it).
    Returns out [Bt, T, Dc], and with return_state the last states [S, Dc, N]
    float32. The last axes are contiguous, other strides are free."""
    cu = cu_seqlens
    try:
        key = ("scan", delta_softplus, sig(u), sig(delta), sig(A), sig(B), sig(C), sig(D), sig(z), sig(delta_bias),
               sig(initial_state), sig(cu))
        lay = plan(key)
    except (AttributeError, TypeError):      # not tensors: the checks say which
        key = lay = None
    if lay is None:
        check_activations("u", u, (3,))
        given = (u, delta, A, B, C, D, z, delta_bias, initial_state, cu_seqlens)
        B, C = _check_scan(u, delta, A, B, C, D, z, delta_bias, u.shape[:2])
        cu, nseq = offsets(cu_seqlens, u.shape[0], u.shape[1], u.device)
        if initial_state is not None:
            check_tensor("initial_state", initial_state, (nseq, *A.shape), torch.float32, u.device)
            initial_state = initial_state.contiguous()
        u, delta, B, C = rows(u), rows(delta), rows(B), rows(C)
        z, A = _opt(z, rows), A.contiguous()
        D, delta_bias = _opt(D, torch.Tensor.contiguous), _opt(delta_bias, torch.Tensor.contiguous)
        lay = _scan_layout(u, delta, A, B, C, z, nseq, int(bool(delta_softplus)))
        if key is not None and all(a is b for a, b in zip(given, (u, delta, A, B, C, D, z, delta_bias, initial_state,
                                                                  cu))):
            _ops.keep_plan(key, lay)
    if wants_grad(u, delta, A, B, C, D, z, delta_bias, initial_state):
        return _SelectiveScan.apply(u, delta, A, B, C, D, z, delta_bias, initial_state, cu, lay, return_state)
    out, state, _ = _scan_forward(lay, u, delta, A, B, C, D, z, delta_bias, initial_state, cu, return_state, False)
    return (out, state) if return_state else out


def selective_scan_step(state, u, delta, A, B, C, D=None, *, z=None, delta_bias=None, delta_softplus: bool = False,
                        slots=None):
    """One token of each request: u, delta, z [Bt, Dc], B and C [Bt, G, N] or [Bt, N];
    returns out [Bt, Dc].

    state [S, Dc, N] float32 (contiguous) is updated in place, in row slots[b] for
    request b (row b without slots, S = Bt). Rows with a negative slot give 0 and touch
    no state; two requests must not share a slot. There is no gradient: inputs that
    require one are refused outside torch.no_grad()."""
    try:
        key = ("scan step", delta_softplus, _ops.sigs(state, u, delta, A, B, C, D, z, delta_bias, slots))
        ints = plan(key)
    except (AttributeError, TypeError):
        key = ints = None
    if ints is None:
        check_activations("u", u, (2,))
        Bt, Dc = u.shape
        dev = u.device
        B, C = _check_scan(u, delta, A, B, C, D, z, delta_bias, (Bt,))
        _check_state("state", state, torch.float32, dev, tuple(A.shape), Bt, slots)
        _ops.check_slots(slots, Bt, dev)
        given = (u, delta, B, C, z, A, D, delta_bias)
        u, delta, B, C = rows(u), rows(delta), rows(B), rows(C)
        z, A = _opt(z, rows), A.contiguous()
        D, delta_bias = _opt(D, torch.Tensor.contiguous), _opt(delta_bias, torch.Tensor.contiguous)
        if any(a is not b for a, b in zip(given, (u, delta, B, C, z, A, D, delta_bias))):
            key = None
        ints = ((DTYPES[u.dtype], int(bool(delta_softplus)), Bt, Dc, A.shape[1], B.shape[1], state.shape[0]),
                (stride(u, 0), stride(delta, 0), 0 if z is None else stride(z, 0), stride(B, 0), stride(B, 1),
                 stride(C, 0), stride(C, 1)), dev.index, _ask_for_gradients(state, u, delta, A, B, C, D, z, delta_bias),
                u.is_contiguous())
        if key is not None:
            _ops.keep_plan(key, ints)
    if ints[3] or forward_ad._current_level >= 0:
        _no_gradients("selective_scan_step", state, u, delta, A, B, C, D, z, delta_bias)
    out = torch.empty_like(u) if ints[4] else _ops.empty(u)
    s32, s64 = (0, 0) if slots is None else _ops.slot_pointers(slots)
    call("pe_selective_scan_step", _SCAN_STEP.pack(
        *ints[0], s32, s64, u.data_ptr(), delta.data_ptr(), 0 if z is None else z.data_ptr(), B.data_ptr(),
        C.data_ptr(), A.data_ptr(), 0 if D is None else D.data_ptr(),
        0 if delta_bias is None else delta_bias.data_ptr(), *ints[1], state.data_ptr(), out.data_ptr()), ints[2])
    increment_version(state)
    return out


# ---- step-by-step references (float64, small sizes) -------------------------------------
def _spans(batch, tokens, cu_seqlens):
    if cu_seqlens is None:
        return [(b, 0, tokens) for b in range(batch)]
    cu = [int(v) for v in (cu_seqlens.tolist() if hasattr(cu_seqlens, "tolist") else cu_seqlens)]
    return [(0, a, b) for a, b in zip(cu, cu[1:])]


def causal_conv_reference(x, weight, bias=None, *, activation=None, initial_state=None, cu_seqlens=None):
    """(out, last states) from the definition, in float64 and differentiable, on any device."""
    W = weight.shape[1]
    x, weight = x.double(), weight.double()
    out, ends = torch.zeros_like(x) + x[:0].sum(), []   # differentiable without sequences too
    for i, (r, a, b) in enumerate(_spans(x.shape[0], x.shape[1], cu_seqlens)):
        head = x.new_zeros(W - 1, x.shape[2]) if initial_state is None else initial_state[i].double()
        seq = torch.cat([head, x[r, a:b]])
        y = sum(weight[:, k] * seq[k:k + b - a] for k in range(W))
        y = y if bias is None else y + bias.double()
        out = out.index_put((torch.tensor(r), torch.arange(a, b)), y * torch.sigmoid(y) if activation else y)
        ends.append(seq[b - a:])
    return out, torch.stack(ends) if ends else x.new_zeros(0, W - 1, x.shape[2])


def selective_scan_reference(u, delta, A, B, C, D=None, *, z=None, delta_bias=None, delta_softplus=False,
                             initial_state=None, cu_seqlens=None):
    """(out, last states) step by step, in float64 and differentiable, on any device."""
    u, delta, A, B, C = (t.double() for t in (u, delta, A, B, C))
    if B.dim() == 3:
        B, C = B.unsqueeze(2), C.unsqueeze(2)
    rep = u.shape[2] // B.shape[2]
    dt = delta if delta_bias is None else delta + delta_bias.double()
    if delta_softplus:
        dt = torch.logaddexp(dt, torch.zeros_like(dt))
    out, ends = torch.zeros_like(u), []
    for i, (r, a, b) in enumerate(_spans(u.shape[0], u.shape[1], cu_seqlens)):
        h = A.new_zeros(A.shape) if initial_state is None else initial_state[i].double()
        ys = []
        for t in range(a, b):
            Bt, Ct = (m[r, t].repeat_interleave(rep, dim=0) for m in (B, C))
            h = torch.exp(dt[r, t, :, None] * A) * h + (dt[r, t] * u[r, t])[:, None] * Bt
            ys.append((h * Ct).sum(-1))
        if ys:
            out = out.index_put((torch.tensor(r), torch.arange(a, b)), torch.stack(ys))
        ends.append(h)
    out = out if D is None else out + D.double() * u
    out = out if z is None else out * z.double() * torch.sigmoid(z.double())
    return out, torch.stack(ends) if ends else A.new_zeros(0, *A.shape)
