"""The recurrent-mixer operators called in other ways than the plain one: empty tensors, states that
change in place, derivatives of other kinds, arguments at the ends of their range, the C entries."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch
from torch.autograd import forward_ad

from pto_einsum import _core, _ops, norm, ssm
from pto_einsum.mixer import SelectiveMixer, contract
from pto_einsum.norm import group_norm, group_norm_reference
from pto_einsum.ssm import (causal_conv, causal_conv_step, selective_scan, selective_scan_reference,
                            selective_scan_step)

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def rand(*shape, seed, dtype=F32, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).to(device)


# ---------------------------------------------------------------------------- empty tensors
def norm_grad_ws_bytes(N, places, C, groups, dtype):
    args = norm._NORM_GRAD.pack(dtype, 0, N, places, C, groups, 1e-5, *[0] * (len(norm._NORM_GRAD.unpack(
        bytes(norm._NORM_GRAD.size))) - 7))
    return _ops.function("pe_group_norm_grad_ws_bytes", ctypes.c_int64, (ctypes.c_char_p,))(args)


EMPTY = [(1000, 0, 64, 4), (2, 0, 4096, 1), (0, 7, 64, 4)]


def test_workspaces_of_empty_norms():
    """In a process of its own: a host that divides by the places of a row ends."""
    here = os.path.dirname(os.path.abspath(__file__))
    code = ("import sys; sys.path[:0] = [%r, %r]\nfrom test_operator_calls import *\n"
            "assert [norm_grad_ws_bytes(*e, dt) for e in EMPTY for dt in (0, 1, 2)] == [0] * 9"
            % (here, os.path.join(os.path.dirname(here), "pto-einsum_b200")))
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert run.returncode == 0, run.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("N,places,C,groups", EMPTY)
def test_gradients_of_empty_norms(N, places, C, groups):
    x, w = rand(N, places, C, seed=1).requires_grad_(), rand(C, seed=2).requires_grad_()
    b = rand(C, seed=3).requires_grad_()
    y = group_norm(x, groups, w, b, activation="silu")
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert dx.shape == x.shape and (dw == 0).all() and (db == 0).all()


# ---------------------------------------------------------------------------- the C entries
def test_a_scan_without_a_place_for_its_output_is_refused():
    """The arguments are checked before anything is launched: no address here is ever used."""
    some = 4096
    args = dict(zip(("dtype", "softplus", "batch", "tokens", "channels", "states", "groups", "nseq"),
                    (1, 1, 2, 10, 16, 16, 1, 2)))
    fields = [*args.values(), 0, some, some, 0, some, some, some, 0, 0, 0, 160, 16, 160, 16, 0, 0, 160, 16, 16, 160, 16, 16]
    call = _ops.function("pe_selective_scan")
    assert call(ssm._SCAN.pack(*fields, 0, 0, 0, 0, 0), None) == 1
    assert _core.core_lib().pe_last_error() == 1


def scan_inputs(B, T, D, N, dt=F32):
    return dict(u=rand(B, T, D, seed=1, dtype=dt), delta=rand(B, T, D, seed=2, dtype=dt), A=-torch.exp(rand(D, N, seed=3)),
                B=rand(B, T, 1, N, seed=4, dtype=dt), C=rand(B, T, 1, N, seed=5, dtype=dt), D=rand(D, seed=6),
                z=rand(B, T, D, seed=7, dtype=dt), delta_bias=rand(D, seed=8) - 2)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_scan_results_at_any_element(dt):
    """Results one element past an aligned address, which a caller of the C entries may choose."""
    B, T, D, N = 2, 70, 48, 16
    k = scan_inputs(B, T, D, N, dt)
    own = {m: t.clone().requires_grad_() for m, t in k.items()}
    y = selective_scan(**own, delta_softplus=True)
    dy = rand(B, T, D, seed=9, dtype=dt)
    want = torch.autograd.grad(y, list(own.values()), dy)
    off = {m: torch.empty(B * T * D + 1, dtype=dt, device="cuda")[1:].view(B, T, D) for m in ("out", "u", "delta", "z")}
    rest = {m: torch.empty_like(k[m]) for m in ("A", "B", "C", "D", "delta_bias")}
    lay = ssm._scan_layout(*(k[m] for m in ("u", "delta", "A", "B", "C", "z")), B, 1)
    ckpt = torch.empty(ssm._core_ckpt(T, B, False, D, N), device="cuda")
    ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")

    def fields(out):
        return ssm._scan_fields(lay, *(k[m] for m in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")), None,
                                None, out, None, ckpt)

    _ops.call("pe_selective_scan", ssm._SCAN.pack(*fields(off["out"]), ws.data_ptr(), ws.numel()), 0)
    assert torch.equal(off["out"], y)
    _ops.call("pe_selective_scan_grad", ssm._SCAN_GRAD.pack(
        *fields(None), 0, 0, dy.data_ptr(), *dy.stride()[:2], 0,
        *(t.data_ptr() for t in (off["u"], off["delta"], off["z"], rest["B"], rest["C"], rest["A"], rest["D"],
                                 rest["delta_bias"])), 0, ws.data_ptr(), ws.numel()), 0)
    for m, g in zip(own, want):
        assert torch.equal(off[m] if m in off else rest[m], g), m


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("shape,groups", [((700, 26000), 1), ((300, 4096), 8), ((4, 3000, 320), 32)])
def test_norm_gradients_with_a_workspace_at_any_float(shape, groups, dt):
    N, C = shape[0], shape[-1]
    t = [rand(*shape, seed=1, dtype=dt), rand(C, seed=2, dtype=dt), rand(C, seed=3, dtype=dt)]
    own = [v.clone().requires_grad_() for v in t]
    y = group_norm(own[0], groups, own[1], own[2], activation="silu")
    dy = rand(*shape, seed=4, dtype=dt)
    want = torch.autograd.grad(y, own, dy)
    places = shape[1] if len(shape) > 2 else 1
    stats = torch.empty(2, N, groups, device="cuda")
    lay = ((norm.DTYPES[dt], 1, N, places, C, groups, 1e-5), (*norm._strides(t[0]), 0, 0), 0)
    got = [torch.empty_like(v) for v in t]
    out = torch.empty_like(t[0])

    def call(name, pack, tail, out):
        fields = (*norm._fields(lay, *t, None, out, stats), *tail)
        n = _ops.sized(name + "_ws_bytes", pack(*fields, 0, 0), 0)
        ws = torch.empty(n // 4 + 1, device="cuda")[1:]
        _ops.call(name, pack(*fields, ws.data_ptr(), n), 0)

    call("pe_group_norm", norm._NORM.pack, (), out)
    call("pe_group_norm_grad", norm._NORM_GRAD.pack, (0, 0, dy.data_ptr(), *norm._strides(dy), got[0].data_ptr(), 0,
                                                      got[1].data_ptr(), got[2].data_ptr()), None)
    # the same sums in another order: a few fp32 roundings, then one to the type
    assert torch.equal(out, y)
    for g, h in zip(got, want):
        off = (g.double() - h.double()).norm() / h.double().norm()
        assert off <= 2 * torch.finfo(dt).eps + 2.0 ** -18, off


# ---------------------------------------------------------------------------- states in place
def token(k, t):
    return {m: v[:, t] if m in ("u", "delta", "B", "C", "z") else v for m, v in k.items()}


@pytest.mark.gpu
def test_a_state_that_a_gradient_still_needs():
    """The steps write through the state's address; autograd has to know."""
    x, w, s = rand(2, 9, 16, seed=1), rand(16, 4, seed=2).requires_grad_(), rand(2, 3, 16, seed=3)
    y = causal_conv(x, w, initial_state=s)
    with torch.no_grad():
        causal_conv_step(x[:, 0], s, w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    k, s = scan_inputs(2, 3, 16, 16), rand(2, 16, 16, seed=9)
    y = (rand(2, 16, 16, seed=10).requires_grad_() * s).sum()
    with torch.no_grad():
        selective_scan_step(s, **token(k, 0), delta_softplus=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        s = torch.zeros(2, 16, 16, device="cuda")
        selective_scan_step(s, **token(k, 0), delta_softplus=True)


@pytest.mark.gpu
def test_scan_gradients_after_the_first_state_went_on():
    """The scan's backward pass starts from its checkpoints: the state itself may be used again."""
    k, got = scan_inputs(2, 9, 16, 16), []
    for change in (False, True):
        s = rand(2, 16, 16, seed=9)
        own = {m: t.clone().requires_grad_() for m, t in k.items()}
        y = selective_scan(**own, initial_state=s, delta_softplus=True)
        if change:
            with torch.no_grad():
                selective_scan_step(s, **token(k, 0), delta_softplus=True)
        got.append(torch.autograd.grad(y.sum(), list(own.values())))
    assert all(torch.equal(a, b) for a, b in zip(*got))


# ---------------------------------------------------------------------------- other derivatives
def test_tangents_are_seen():
    x = torch.ones(3)
    assert not _ops.wants_grad(x, None)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        with torch.no_grad():
            assert _ops.wants_grad(None, x, dual) and not _ops.wants_grad(x, None)


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [True, False])
def test_forward_derivatives_are_refused(grad):
    """The operators have none: torch's error for that, not an output without a tangent."""
    x, w, k = rand(2, 9, 16, seed=1), rand(16, 4, seed=2), scan_inputs(2, 9, 16, 16)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for f in (lambda: causal_conv(dual, w), lambda: selective_scan(**{**k, "u": dual}, delta_softplus=True),
                  lambda: group_norm(dual, 4), lambda: group_norm(x, 4, gate=dual)):
            with pytest.raises(NotImplementedError, match="jvp"):
                f()
        causal_conv(x, w)


@pytest.mark.gpu
def test_steps_refuse_gradients():
    """Their outputs carry none: an input that asks for one, or has a tangent, is an error."""
    x, w, k = rand(2, 16, seed=1), rand(16, 4, seed=2), token(scan_inputs(2, 1, 16, 16), 0)
    cs, ss = rand(2, 3, 16, seed=3), rand(2, 16, 16, seed=4)
    before = cs.clone(), ss.clone()
    for a in ((x.clone().requires_grad_(), w), (x, w.clone().requires_grad_())):
        with pytest.raises(ValueError, match="no gradient"):
            causal_conv_step(a[0], cs, a[1])
    for m in k:
        with pytest.raises(ValueError, match="no gradient"):
            selective_scan_step(ss, **{**k, m: k[m].clone().requires_grad_()})
    with torch.no_grad(), forward_ad.dual_level(), pytest.raises(ValueError, match="no gradient"):
        causal_conv_step(forward_ad.make_dual(x, x.clone()), cs, w)
    assert torch.equal(cs, before[0]) and torch.equal(ss, before[1])
    with torch.no_grad():
        causal_conv_step(x, cs, w.clone().requires_grad_())


# ---------------------------------------------------------------------------- ends of the range
@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF16])
def test_norms_of_large_finite_maps(dt):
    """Means past 1.8e19, whose squares fp32 does not hold, in maps that are read in chunks. The
    deviations, 1e-3 of the mean, are known to 2^-24 of it."""
    N, S, C, G = 16, 2100, 320, 32
    x = torch.full((N, S, C), 2e19, device="cuda").to(dt)
    if dt == F32:
        x = x * (1 + 1e-3 * rand(N, S, C, seed=1))
    n0 = _core.launch_count()
    y = group_norm(x, G)
    assert _core.launch_count() == n0 + 3            # sums of the chunks, their joining, the result
    r = group_norm_reference(x, G)
    if dt == F32:
        assert ((y - r).norm() / r.norm()).item() <= 1000 * 2.0 ** -24 + 2.0 ** -20
    else:
        assert (y == 0).all()


# ---------------------------------------------------------------------------- second derivatives
class Detached:
    """A backend whose results know no gradient, as the compiled runners' do not."""

    def contract(self, eq, a, b):
        return torch.einsum(eq, a.detach(), b.detach())


def test_second_derivatives_of_contractions():
    a = rand(2, 3, 4, seed=1, device="cpu").double().requires_grad_()
    b = rand(4, 5, seed=2, device="cpu").double().requires_grad_()
    g = rand(2, 3, 5, seed=3, device="cpu").double()

    def second(f):
        y = f("bte,ef->btf", a, b)
        da, db = torch.autograd.grad((y * y * g).sum(), (a, b), create_graph=True)
        return torch.autograd.grad((da ** 3).sum() + (db ** 2).sum(), (a, b))

    for u, v in zip(second(lambda eq, a, b: contract(Detached(), eq, a, b)), second(torch.einsum)):
        assert torch.allclose(u, v, rtol=1e-12)


@pytest.mark.gpu
def test_second_derivatives_of_the_layer_are_refused():
    """Its other operators have first derivatives only, and say so."""
    mix = SelectiveMixer(32, 64, heads=2, dtype=F32, device="cuda", seed=3, requires_grad=True)
    y = mix(rand(2, 24, 32, seed=1))
    d, = torch.autograd.grad((y * y).sum(), mix.params["w_in"], create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (d * d).sum().backward()
    mix.cleanup()


# ---------------------------------------------------------------------------- offsets
@pytest.mark.gpu
def test_offsets_past_32_bits_are_reported():
    """64-bit offsets whose low halves would make a table."""
    x, w = rand(1, 10, 16, seed=1), rand(16, 4, seed=2)
    assert _core.device_error() == 0
    for cu in ([0, 2 ** 32 + 5, 10], [2 ** 32, 5, 10], [0, 5, 10 - 2 ** 32], [0, 5, 2 ** 32 + 10]):
        causal_conv(x, w, cu_seqlens=torch.tensor(cu, device="cuda"))
        assert _core.device_error() & 0xFF == 1, cu
    causal_conv(x, w, cu_seqlens=torch.tensor([0, 5, 10], device="cuda"))
    assert _core.device_error() == 0


def test_host_offsets_are_whole_numbers():
    cpu = torch.device("cpu")
    for cu in ([0, 2.5, 4], torch.tensor([0.0, 2.5, 4.0])):
        with pytest.raises(ValueError, match="whole numbers"):
            _ops.offsets(cu, 1, 4, cpu)
    for cu in ([0, 2, 4], (0, 2, 4), torch.tensor([0, 2, 4]), torch.tensor([0, 2, 4]).numpy(), range(0, 6, 2),
               [torch.tensor(0), torch.tensor(2), torch.tensor(4)]):
        table, n = _ops.offsets(cu, 1, 4, cpu)
        assert table.tolist() == [0, 2, 4] and n == 2


# ---------------------------------------------------------------------------- infinite rates
@pytest.mark.gpu
@pytest.mark.parametrize("B,T,D", [(2, 20, 16), (1, 5000, 48)])
def test_states_that_forget_everything(B, T, D):
    """A = -inf: each token starts from nothing, and the last state is its own. A tile's rows past the
    last token, whose steps are zero, must not take part. Whole sequences and one split along time."""
    k = scan_inputs(B, T, D, 16)
    k["A"][:, 3] = -float("inf")
    y, end = selective_scan(**k, delta_softplus=True, return_state=True)
    r, rend = selective_scan_reference(**k, delta_softplus=True)
    tol = 2.0 ** -20 + T ** 0.5 * 2.0 ** -18
    for a, b in ((y, r), (end, rend)):
        assert torch.isfinite(a).all() and ((a - b).norm() / b.norm()).item() <= tol
    # the gradients are those of a rate so large that it forgets as well
    got = []
    for rate in (-float("inf"), -1e30):
        own = {m: t.clone().requires_grad_() for m, t in k.items()}
        with torch.no_grad():
            own["A"][:, 3] = rate
        y, end = selective_scan(**own, delta_softplus=True, return_state=True)
        got.append(torch.autograd.grad([y, end], list(own.values()), [torch.ones_like(y), torch.ones_like(end)]))
    for m, a, b in zip(k, *got):
        assert torch.isfinite(a).all() and torch.equal(a, b), m


# ---------------------------------------------------------------------------- shared memory
@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("N", [1, 6, 7, 8, 9, 11, 12, 40])
def test_split_scans_of_any_number_of_states(N, dt):
    """The launches' shared memory grows with the states, past what a block has without asking for more."""
    k = scan_inputs(1, 600, 40, N, dt)
    k["delta_bias"] = k["delta_bias"] - 2
    own = {m: t.clone().requires_grad_() for m, t in k.items()}
    ref = {m: t.double().requires_grad_() for m, t in k.items()}
    n0 = _core.launch_count()
    y, r = selective_scan(**own, delta_softplus=True), selective_scan_reference(**ref, delta_softplus=True)[0]
    assert _core.launch_count() == n0 + 3
    dy = rand(*y.shape, seed=9, dtype=dt)
    got = torch.autograd.grad(y, list(own.values()), dy)
    assert _core.launch_count() == n0 + 8
    want = torch.autograd.grad(r, list(ref.values()), dy.double())
    for m, a, b in zip(k, got, want):
        unit = torch.finfo(a.dtype).eps / 2
        tol = 4 * (unit + 2.0 ** -20 + 600 ** 0.5 * 2.0 ** -18)
        assert torch.isfinite(a).all() and ((a - b).norm() / b.norm()).item() <= tol, m
