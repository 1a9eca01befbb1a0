"""Causal convolution and selective scan (pto_einsum.ssm) against their definitions in
float64: prompts, packed sequences, single tokens, gradients, refusals.

Tolerances (relative 2-norm), derived from the arithmetic: an output rounded once has an
error of at most its type's unit roundoff u. A state is multiplied once a token by an
exponential good to 2^-22 of an argument rounded twice, and added to with one rounding,
so its error grows by at most 2^-21 a token it remembers; the convolution's fixed sum of
a few terms stays below 2^-20. Gradients pass through the recurrence twice and add
products of two such quantities: four times that."""
import subprocess

import pytest
import torch

from pto_einsum import INCLUDE_DIR, _core, norm, ssm
from pto_einsum.ssm import (causal_conv, causal_conv_reference, causal_conv_step, selective_scan,
                            selective_scan_reference, selective_scan_step)

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ROUND = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
STEP, FIXED = 2.0 ** -21, 2.0 ** -20


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    assert a.shape == b.shape, (a.shape, b.shape)
    assert torch.isfinite(a).all() == torch.isfinite(b).all()
    if not b.numel():
        return 0.0
    off, size = (a - b).norm().item(), b.norm().item()
    return off / size if size else off


def rand(*shape, seed, dtype=F32, scale=1.0, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(device)


# ---------------------------------------------------------------------------- CPU
def test_argument_structs_match_the_header(tmp_path):
    names = {"pe_scan_args": ssm._SCAN, "pe_scan_grad_args": ssm._SCAN_GRAD, "pe_scan_step_args": ssm._SCAN_STEP,
             "pe_conv_args": ssm._CONV, "pe_conv_grad_args": ssm._CONV_GRAD, "pe_conv_step_args": ssm._CONV_STEP,
             "pe_norm_args": norm._NORM, "pe_norm_grad_args": norm._NORM_GRAD}
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "pto_einsum_b200.h"\nint main(void) {\n'
                   + "".join(f'printf("%zu\\n", sizeof({n}));\n' for n in names) + "return 0; }\n")
    exe = str(tmp_path / "sizes")
    subprocess.run(["gcc", "-I", INCLUDE_DIR, str(src), "-o", exe], check=True)
    sizes = subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()
    assert [int(s) for s in sizes] == [p.size for p in names.values()]


def test_host_tensors_are_refused():
    x, w = torch.zeros(1, 4, 8), torch.zeros(8, 4)
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        causal_conv(x, w)
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        selective_scan(x, x, torch.zeros(8, 16), torch.zeros(1, 4, 16), torch.zeros(1, 4, 16))


@pytest.mark.parametrize("cu", [[0, 5, 5, 9], None])
def test_references_continue_from_their_states(cu):
    x, w, b = rand(1, 9, 6, seed=1), rand(6, 4, seed=2), rand(6, seed=3)
    y, end = causal_conv_reference(x, w, b, activation="silu", cu_seqlens=cu)
    if cu is None:
        y1, mid = causal_conv_reference(x[:, :4], w, b, activation="silu")
        y2, fin = causal_conv_reference(x[:, 4:], w, b, activation="silu", initial_state=mid)
        assert torch.equal(torch.cat([y1, y2], 1), y) and torch.equal(fin, end)
    else:
        for s, (a, e) in enumerate(zip(cu, cu[1:])):
            one, last = causal_conv_reference(x[:, a:e], w, b, activation="silu")
            assert torch.equal(one, y[:, a:e]) and torch.equal(last[0], end[s])


def test_scan_reference_is_the_closed_form():
    """h_t = sum_s exp(A (S_t - S_s)) dt_s u_s B_s with S the running sum of dt."""
    u, d, A = rand(1, 7, 3, seed=1), rand(1, 7, 3, seed=2).abs(), -rand(3, 5, seed=3).abs()
    B, C = rand(1, 7, 5, seed=4), rand(1, 7, 5, seed=5)
    y, _ = selective_scan_reference(u, d, A, B, C)
    S = d.double().cumsum(1)[0]
    t = torch.arange(7)
    e = torch.exp(A.double() * (S[:, None] - S[None])[..., None]) * (t[:, None] >= t[None])[..., None, None]
    h = (e * ((d.double() * u.double())[0, None, ..., None] * B[0, None, :, None].double())).sum(1)
    assert rel(y[0], (h * C[0, :, None].double()).sum(-1)) < 1e-14


# ---------------------------------------------------------------------------- GPU helpers
def gpu():
    return torch.device("cuda", 0)


LAYOUTS = ["plain", "columns", "time-major"]


def laid_out(x, layout):
    """The same values in another memory layout (channels stay contiguous)."""
    if layout == "columns":                      # a slice of wider rows, off the 16-byte boundary
        wide = torch.full((*x.shape[:-1], x.shape[-1] + 5), float("nan"), dtype=x.dtype, device=x.device)
        wide[..., 3:3 + x.shape[-1]] = x
        return wide[..., 3:3 + x.shape[-1]]
    if layout == "time-major" and x.dim() > 2:
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    return x


def compare_grads(got, want, names, dtypes, tol):
    for name, a, b, dt in zip(names, got, want, dtypes):
        assert a.dtype == dt, (name, a.dtype)
        assert rel(a, b) <= tol + 4 * ROUND[dt], (name, rel(a, b), tol)


# ---------------------------------------------------------------------------- convolution
CONV = [  # B, T, C, W, cu, init
    (1, 1, 8, 4, None, False), (2, 3, 64, 4, None, True), (3, 17, 24, 3, None, False), (2, 130, 40, 2, None, True),
    (1, 0, 16, 4, None, True), (0, 5, 16, 4, None, False), (2, 33, 7, 4, None, True), (1, 40, 264, 4, [0, 0, 1, 3, 20, 20, 40], True),
    (1, 97, 33, 3, [0, 50, 97, 97], False), (1, 64, 128, 4, [0, 16, 32, 48, 64], True)]


def conv_inputs(B, T, C, W, cu, init, dt, layout="plain", seed=0):
    n = len(cu) - 1 if cu else B
    x = laid_out(rand(B, T, C, seed=seed + 1, dtype=dt, device=gpu()), layout)
    return (x, rand(C, W, seed=seed + 2, dtype=dt, scale=W ** -0.5, device=gpu()),
            rand(C, seed=seed + 3, dtype=dt, device=gpu()),
            rand(n, W - 1, C, seed=seed + 4, dtype=dt, device=gpu()) if init else None)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("B,T,C,W,cu,init", CONV)
def test_conv_forward(B, T, C, W, cu, init, layout, dt):
    x, w, b, i = conv_inputs(B, T, C, W, cu, init, dt, layout)
    n0 = _core.launch_count()
    for act, bias in (("silu", b), (None, None)):
        y, end = causal_conv(x, w, bias, activation=act, initial_state=i, cu_seqlens=cu, return_state=True)
        r, rend = causal_conv_reference(x, w, bias, activation=act, initial_state=i, cu_seqlens=cu)
        assert y.dtype == dt and y.is_contiguous()
        assert rel(y, r) <= ROUND[dt] + FIXED
        assert torch.equal(end.double(), rend)        # copies of inputs
    assert _core.launch_count() > n0 or B * T == 0
    assert _core.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("B,T,C,W,cu,init", CONV)
def test_conv_gradients(B, T, C, W, cu, init, layout, dt):
    x, w, b, i = conv_inputs(B, T, C, W, cu, init, dt, layout)
    n = len(cu) - 1 if cu else B
    dy, dend = rand(B, T, C, seed=8, dtype=dt, device=gpu()), rand(n, W - 1, C, seed=9, dtype=dt, device=gpu())
    leaves = [t for t in (x, w, b, i) if t is not None]
    own = [t.detach().requires_grad_() for t in leaves]
    ref = [t.detach().double().requires_grad_() for t in leaves]
    for act in ("silu", None):
        y, end = causal_conv(*own[:3], activation=act, initial_state=own[3] if init else None, cu_seqlens=cu,
                             return_state=True)
        got = torch.autograd.grad([y, end], own, [laid_out(dy, layout), dend])
        r, rend = causal_conv_reference(*ref[:3], activation=act, initial_state=ref[3] if init else None,
                                        cu_seqlens=cu)
        want = torch.autograd.grad([r, rend] if B else [r], ref, [dy.double(), dend.double()] if B else [dy.double()],
                                   allow_unused=True)
        want = [torch.zeros_like(t) if g is None else g for g, t in zip(want, ref)]
        compare_grads(got, want, ("x", "weight", "bias", "initial_state"), [dt] * 4, 4 * FIXED)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("C,W", [(64, 4), (9, 3)])
def test_conv_pieces_and_tokens_are_the_whole(C, W, dt):
    """A prompt in pieces, then token by token from the state, gives the whole prompt's bits."""
    x, w, b, _ = conv_inputs(2, 41, C, W, None, False, dt)
    y, end = causal_conv(x, w, b, activation="silu", return_state=True)
    y1, state = causal_conv(x[:, :30], w, b, activation="silu", return_state=True)
    assert torch.equal(y1, y[:, :30])
    y2, state = causal_conv(x[:, 30:35], w, b, activation="silu", initial_state=state, return_state=True)
    assert torch.equal(y2, y[:, 30:35])
    pool = torch.full((5, W - 1, C), float("nan"), dtype=dt, device=gpu())
    slots = torch.tensor([4, 1], dtype=torch.int32, device=gpu())
    pool[slots.long()] = state
    for t in range(35, 41):
        assert torch.equal(causal_conv_step(x[:, t], pool, w, b, activation="silu", slots=slots), y[:, t])
    assert torch.equal(pool[slots.long()], end)
    assert torch.isnan(pool[[0, 2, 3]]).all()


# ---------------------------------------------------------------------------- scan
SCAN = [  # B, T, D, N, G, cu, gate, skip, init
    (1, 1, 8, 16, 1, None, True, True, False), (2, 16, 40, 16, 1, None, True, True, True),
    (2, 17, 33, 16, 1, None, False, False, False), (1, 100, 64, 5, 2, None, True, True, True),
    (2, 31, 21, 24, 3, None, True, False, True), (1, 40, 6, 3, 2, None, False, True, True),
    (1, 50, 20, 33, 1, None, True, True, False), (2, 33, 12, 128, 2, None, True, True, True),
    (1, 0, 8, 16, 1, None, True, True, True), (0, 4, 8, 16, 1, None, True, True, False),
    (1, 90, 37, 16, 1, [0, 0, 1, 17, 33, 33, 90, 90], True, True, True), (1, 64, 16, 8, 1, [0, 32, 64], False, True, False),
    (1, 300, 132, 16, 1, None, True, True, False), (1, 64, 70, 7, 1, [0, 16, 64], True, True, True)]


def scan_inputs(B, T, D, N, G, cu, gate, skip, init, dt, layout="plain", seed=0):
    n = len(cu) - 1 if cu else B
    dev = gpu()

    def act(*shape, seed):
        return laid_out(rand(*shape, seed=seed, dtype=dt, device=dev), layout)

    k = dict(u=act(B, T, D, seed=seed + 1), delta=act(B, T, D, seed=seed + 2),
             A=-torch.exp(rand(D, N, seed=seed + 3)).to(dev), B=act(B, T, G, N, seed=seed + 4),
             C=act(B, T, G, N, seed=seed + 5), D=rand(D, seed=seed + 6, device=dev) if skip else None,
             z=act(B, T, D, seed=seed + 7) if gate else None, delta_bias=rand(D, seed=seed + 8, device=dev) - 2,
             initial_state=rand(n, D, N, seed=seed + 9, device=dev) if init else None)
    return k


def leaves_of(k):
    return [name for name, t in k.items() if t is not None]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("B,T,D,N,G,cu,gate,skip,init", SCAN)
def test_scan_forward(B, T, D, N, G, cu, gate, skip, init, layout, dt):
    k = scan_inputs(B, T, D, N, G, cu, gate, skip, init, dt, layout)
    y, end = selective_scan(**k, delta_softplus=True, cu_seqlens=cu, return_state=True)
    r, rend = selective_scan_reference(**k, delta_softplus=True, cu_seqlens=cu)
    assert y.dtype == dt and y.is_contiguous() and end.dtype == F32
    assert rel(y, r) <= ROUND[dt] + FIXED + T * STEP
    assert rel(end, rend) <= FIXED + T * STEP
    assert torch.equal(y, selective_scan(**k, delta_softplus=True, cu_seqlens=cu))
    assert _core.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("B,T,D,N,G,cu,gate,skip,init", SCAN)
def test_scan_gradients(B, T, D, N, G, cu, gate, skip, init, layout, dt):
    k = scan_inputs(B, T, D, N, G, cu, gate, skip, init, dt, layout)
    names = leaves_of(k)
    n = len(cu) - 1 if cu else B
    own = {m: t.detach().requires_grad_() if t is not None else None for m, t in k.items()}
    ref = {m: t.detach().double().requires_grad_() if t is not None else None for m, t in k.items()}
    dy, dend = rand(B, T, D, seed=20, dtype=dt, device=gpu()), rand(n, D, N, seed=21, device=gpu())
    y, end = selective_scan(**own, delta_softplus=True, cu_seqlens=cu, return_state=True)
    got = torch.autograd.grad([y, end], [own[m] for m in names], [laid_out(dy, layout), dend], retain_graph=True)
    r, rend = selective_scan_reference(**ref, delta_softplus=True, cu_seqlens=cu)
    want = torch.autograd.grad([r, rend] if B else [r], [ref[m] for m in names],
                               [dy.double(), dend.double()] if B else [dy.double()], allow_unused=True)
    want = [torch.zeros_like(ref[m]) if g is None else g for g, m in zip(want, names)]
    compare_grads(got, want, names, [k[m].dtype for m in names], 4 * (FIXED + T * STEP))
    again = torch.autograd.grad([y, end], [own[m] for m in names], [laid_out(dy, layout), dend])
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.gpu
def test_scan_gradients_against_differences():
    """Central differences of the float64 definition along random directions."""
    k = scan_inputs(1, 40, 12, 16, 2, [0, 15, 40], True, True, True, F32)
    names = leaves_of(k)
    own = {m: t.detach().requires_grad_() for m, t in k.items()}
    dy = rand(1, 40, 12, seed=30, device=gpu())
    got = dict(zip(names, torch.autograd.grad(
        selective_scan(**own, delta_softplus=True, cu_seqlens=[0, 15, 40]), [own[m] for m in names], dy)))
    eps = 1e-5
    for i, m in enumerate(names):
        v = rand(*k[m].shape, seed=40 + i, device=gpu()).double()
        f = [(selective_scan_reference(**{**k, m: k[m].double() + s * eps * v}, delta_softplus=True,
                                       cu_seqlens=[0, 15, 40])[0] * dy).sum().item() for s in (1, -1)]
        want, have = (f[0] - f[1]) / (2 * eps), (got[m].double() * v).sum().item()
        # the differences' own error is of order eps^2 f'''; the gradient's as in the test above,
        # with the size of a sum of its terms in place of the sum
        size = (got[m].double() * v).norm().item()
        assert abs(want - have) <= 1e-6 * abs(want) + 4 * (FIXED + 40 * STEP) * 40 * size, (m, want, have)


@pytest.mark.gpu
def test_conv_gradients_against_differences():
    x, w, b, i = conv_inputs(1, 40, 12, 4, [0, 15, 40], True, F32)
    t = dict(x=x, weight=w, bias=b, initial_state=i)
    own = {m: v.detach().requires_grad_() for m, v in t.items()}
    dy = rand(1, 40, 12, seed=30, device=gpu())
    got = dict(zip(t, torch.autograd.grad(
        causal_conv(**own, activation="silu", cu_seqlens=[0, 15, 40]), list(own.values()), dy)))
    eps = 1e-5
    for j, m in enumerate(t):
        v = rand(*t[m].shape, seed=40 + j, device=gpu()).double()
        f = [(causal_conv_reference(**{**t, m: t[m].double() + s * eps * v}, activation="silu",
                                    cu_seqlens=[0, 15, 40])[0] * dy).sum().item() for s in (1, -1)]
        want, have = (f[0] - f[1]) / (2 * eps), (got[m].double() * v).sum().item()
        size = (got[m].double() * v).norm().item()
        assert abs(want - have) <= 1e-6 * abs(want) + 4 * FIXED * 40 * size, (m, want, have)


@pytest.mark.gpu
@pytest.mark.parametrize("delta,bias", [(-30.0, 0.0), (30.0, 0.0), (0.0, 60.0), (-90.0, -20.0)])
def test_scan_with_extreme_step_sizes(delta, bias):
    """Steps of nothing (the state stays) and of 30 to 60 (the state is forgotten at once)."""
    k = scan_inputs(1, 40, 16, 16, 1, None, True, True, True, F32)
    k["delta"] = torch.full_like(k["delta"], delta)
    k["delta_bias"] = torch.full_like(k["delta_bias"], bias)
    y, end = selective_scan(**k, delta_softplus=True, return_state=True)
    r, rend = selective_scan_reference(**k, delta_softplus=True)
    # an argument of size |x| rounded to 24 bits moves its exponential by |x| 2^-24: 90 of the
    # softplus on top of the steps' own error
    assert rel(y, r) <= FIXED + 40 * STEP + 110 * 2.0 ** -24
    assert rel(end, rend) <= FIXED + 40 * STEP + 110 * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("softplus", [False, True])
def test_scan_without_bias_and_softplus(softplus):
    k = scan_inputs(2, 50, 24, 16, 1, None, False, False, False, F32)
    k["delta"], k["delta_bias"] = k["delta"].abs(), None
    k["B"], k["C"] = k["B"][:, :, 0], k["C"][:, :, 0]        # one group without its axis
    own = {m: t.detach().requires_grad_() if t is not None else None for m, t in k.items()}
    ref = {m: t.detach().double().requires_grad_() if t is not None else None for m, t in k.items()}
    y, r = selective_scan(**own, delta_softplus=softplus), selective_scan_reference(**ref, delta_softplus=softplus)[0]
    assert rel(y, r) <= FIXED + 50 * STEP
    names = leaves_of(k)
    dy = rand(*y.shape, seed=5, device=gpu())
    got = torch.autograd.grad(y, [own[m] for m in names], dy)
    want = torch.autograd.grad(r, [ref[m] for m in names], dy.double())
    compare_grads(got, want, names, [F32] * len(names), 4 * (FIXED + 50 * STEP))


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,D,N,cu", [(1, 5000, 48, 16, None), (2, 3001, 20, 5, None),
                                        (1, 6000, 32, 16, [0, 2500, 2500, 2600, 6000])])
def test_scan_of_long_prompts(B, T, D, N, cu):
    """Few channels and many tokens: the time axis is split over blocks."""
    k = scan_inputs(B, T, D, N, 1, cu, True, True, True, F32)
    k["delta_bias"] = k["delta_bias"] - 2      # longer memories
    y, end = selective_scan(**k, delta_softplus=True, cu_seqlens=cu, return_state=True)
    r, rend = selective_scan_reference(**k, delta_softplus=True, cu_seqlens=cu)
    # a state remembers at most T tokens, but errors of so many differ in sign: their root
    assert rel(y, r) <= FIXED + T ** 0.5 * 8 * STEP
    assert rel(end, rend) <= FIXED + T ** 0.5 * 8 * STEP
    names = leaves_of(k)
    own = {m: t.detach().requires_grad_() for m, t in k.items()}
    dy = rand(*y.shape, seed=5, device=gpu())
    y2 = selective_scan(**own, delta_softplus=True, cu_seqlens=cu)
    assert rel(y2, r) <= FIXED + T ** 0.5 * 8 * STEP
    got = torch.autograd.grad(y2, [own[m] for m in names], dy)
    ref = {m: t.detach().double().requires_grad_() for m, t in k.items()}
    want = torch.autograd.grad(selective_scan_reference(**ref, delta_softplus=True, cu_seqlens=cu)[0],
                               [ref[m] for m in names], dy.double())
    compare_grads(got, want, names, [F32] * len(names), 4 * (FIXED + T ** 0.5 * 8 * STEP))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("D,N,G,layout", [(64, 16, 1, "plain"), (33, 5, 3, "columns"), (20, 128, 2, "plain"),
                                          (9, 24, 1, "columns"), (130, 1, 1, "plain")])
def test_scan_tokens_continue_a_prompt(D, N, G, layout, dt):
    k = scan_inputs(2, 20, D, N, G, None, True, True, True, dt, layout)
    kw = dict(delta_softplus=True)
    y, end = selective_scan(**k, **kw, return_state=True)
    per = ("u", "delta", "B", "C", "z")
    k1 = {m: t[:, :12] if m in per else t for m, t in k.items()}
    y1, mid = selective_scan(**k1, **kw, return_state=True)
    assert rel(y1, y[:, :12]) <= ROUND[dt] + FIXED
    pool = torch.full((6, D, N), float("nan"), device=gpu())
    slots = torch.tensor([5, 2], device=gpu())           # int64
    pool[slots] = mid
    rest = {m: k[m] for m in ("A", "D", "delta_bias")}
    for t in range(12, 20):
        yt = selective_scan_step(pool, k["u"][:, t], k["delta"][:, t], B=k["B"][:, t], C=k["C"][:, t], z=k["z"][:, t],
                                 **rest, **kw, slots=slots)
        assert rel(yt, y[:, t]) <= 2 * ROUND[dt] + FIXED + 20 * STEP
    assert rel(pool[slots], end) <= FIXED + 20 * STEP
    assert torch.isnan(pool[[0, 1, 3, 4]]).all()
    state = mid.clone()                                   # without slots
    yt = selective_scan_step(state, k["u"][:, 12], k["delta"][:, 12], B=k["B"][:, 12], C=k["C"][:, 12],
                             z=k["z"][:, 12], **rest, **kw)
    assert rel(yt, y[:, 12]) <= 2 * ROUND[dt] + FIXED + 20 * STEP


@pytest.mark.gpu
def test_steps_skip_negative_slots_and_report_wrong_ones():
    dev = gpu()
    k = scan_inputs(4, 1, 16, 16, 1, None, True, True, False, F16)
    one = {m: k[m][:, 0] for m in ("u", "delta", "B", "C", "z")}
    rest = {m: k[m] for m in ("A", "D", "delta_bias")}
    pool = rand(3, 16, 16, seed=3, device=dev)
    before = pool.clone()
    assert _core.device_error() == 0
    y = selective_scan_step(pool, **one, **rest, slots=torch.tensor([1, -1, 0, -7], device=dev))
    assert (y[[1, 3]] == 0).all() and torch.equal(pool[2], before[2]) and not torch.equal(pool[:2], before[:2])
    assert _core.device_error() == 0
    selective_scan_step(pool, **one, **rest, slots=torch.tensor([-1, 3, -1, -1], device=dev))
    assert _core.device_error() & 0xFF == 1 and _core.device_error() == 0
    x, w = rand(4, 16, seed=1, dtype=F16, device=dev), rand(16, 4, seed=2, dtype=F16, device=dev)
    cpool = rand(3, 3, 16, seed=4, dtype=F16, device=dev)
    cbefore = cpool.clone()
    y = causal_conv_step(x, cpool, w, slots=torch.tensor([-1, 2, -1, 9], dtype=torch.int32, device=dev))
    assert (y[[0, 2, 3]] == 0).all() and torch.equal(cpool[:2], cbefore[:2])
    assert _core.device_error() & 0xFF == 1 and _core.device_error() == 0


@pytest.mark.gpu
def test_offsets_on_the_device_and_wrong_ones():
    x, w, b, i = conv_inputs(1, 40, 64, 4, [0, 5, 5, 40], True, F16)
    k = scan_inputs(1, 40, 16, 16, 1, [0, 5, 5, 40], True, True, True, F16)
    for dtype in (torch.int32, torch.int64):
        cu = torch.tensor([0, 5, 5, 40], dtype=dtype, device=gpu())
        assert torch.equal(causal_conv(x, w, b, initial_state=i, cu_seqlens=cu),
                           causal_conv(x, w, b, initial_state=i, cu_seqlens=[0, 5, 5, 40]))
        assert torch.equal(selective_scan(**k, delta_softplus=True, cu_seqlens=cu),
                           selective_scan(**k, delta_softplus=True, cu_seqlens=[0, 5, 5, 40]))
    assert _core.device_error() == 0
    # wrong tables stay inside the tensors and are reported
    for bad in ([0, 30, 5, 40], [0, 5, 5, 39], [-4, 5, 5, 90], [3, 5, 5, 40]):
        cu = torch.tensor(bad, dtype=torch.int32, device=gpu())
        causal_conv(x, w, b, initial_state=i, cu_seqlens=cu, return_state=True)
        assert _core.device_error() & 0xFF == 1
        selective_scan(**k, delta_softplus=True, cu_seqlens=cu, return_state=True)
        assert _core.device_error() & 0xFF == 1
    assert _core.device_error() == 0


@pytest.mark.gpu
def test_infinities_stay_in_their_sequence():
    cu = [0, 20, 41, 60]
    x, w, b, i = conv_inputs(1, 60, 16, 4, cu, True, F32)
    k = scan_inputs(1, 60, 16, 16, 1, cu, True, True, True, F32)
    sp = dict(delta_softplus=True, cu_seqlens=cu)
    y0, s0 = causal_conv(x, w, b, initial_state=i, cu_seqlens=cu), selective_scan(**k, **sp)
    x2, k2 = x.clone(), dict(k, u=k["u"].clone())
    x2[:, 30], k2["u"][:, 30] = float("nan"), float("inf")
    y1, s1 = causal_conv(x2, w, b, initial_state=i, cu_seqlens=cu), selective_scan(**k2, **sp)
    keep = [t for t in range(60) if not 30 <= t < 41]
    assert torch.equal(y0[:, keep], y1[:, keep]) and torch.equal(s0[:, keep], s1[:, keep])
    assert not torch.isfinite(s1[:, 30:41]).any() and torch.isnan(y1[:, 30:34]).all()
    assert torch.equal(y0[:, 34:], y1[:, 34:])


@pytest.mark.gpu
def test_row_strides_past_32_bits():
    """Two rows of tokens 2^31 elements apart."""
    dev, far = gpu(), 2 ** 31 + 64
    buf = torch.empty(far + 40 * 64, dtype=F16, device=dev)
    x = buf.as_strided((2, 40, 64), (far, 64, 1))
    x.copy_(rand(2, 40, 64, seed=1, dtype=F16, device=dev))
    w = rand(64, 4, seed=2, dtype=F16, device=dev)
    assert torch.equal(causal_conv(x, w), causal_conv(x.contiguous(), w))
    k = scan_inputs(2, 40, 64, 16, 1, None, False, True, False, F16)
    assert torch.equal(selective_scan(**{**k, "u": x}, delta_softplus=True),
                       selective_scan(**{**k, "u": x.contiguous()}, delta_softplus=True))


@pytest.mark.gpu
def test_other_streams_and_graphs():
    k = scan_inputs(1, 200, 64, 16, 1, None, True, True, False, F16)
    x, w, b, _ = conv_inputs(1, 200, 64, 4, None, False, F16)
    y0, c0 = selective_scan(**k, delta_softplus=True), causal_conv(x, w, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y1, c1 = selective_scan(**k, delta_softplus=True), causal_conv(x, w, b)
    s.synchronize()
    assert torch.equal(y0, y1) and torch.equal(c0, c1)
    one = {m: k[m][:, 0] for m in ("u", "delta", "B", "C", "z")}
    rest = dict({m: k[m] for m in ("A", "D", "delta_bias")}, delta_softplus=True)
    state, cs = torch.zeros(1, 64, 16, device=gpu()), torch.zeros(1, 3, 64, dtype=F16, device=gpu())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cy = causal_conv_step(x[:, 0], cs, w, b)
        y = selective_scan_step(state, **one, **rest)
    for t in range(3):
        g.replay()
    state2, cs2 = torch.zeros_like(state), torch.zeros_like(cs)
    for t in range(3):
        cy2 = causal_conv_step(x[:, 0], cs2, w, b)
        y2 = selective_scan_step(state2, **one, **rest)
    assert torch.equal(state, state2) and torch.equal(cs, cs2) and torch.equal(y, y2) and torch.equal(cy, cy2)


@pytest.mark.gpu
def test_refusals():
    dev = gpu()
    x, w, b, i = conv_inputs(2, 10, 16, 4, None, True, F16)
    k = scan_inputs(2, 10, 16, 16, 1, None, True, True, True, F16)

    def no(error, match, f, *a, **kw):
        with pytest.raises(error, match=match):
            f(*a, **kw)

    no(ValueError, "width of 2 to 4", causal_conv, x, rand(16, 5, seed=1, dtype=F16, device=dev))
    no(TypeError, "weight must be", causal_conv, x, w.float())
    no(TypeError, "float32, float16 or bfloat16", causal_conv, x.double(), w.double())
    no(ValueError, "bias must have shape", causal_conv, x, w, b[:8])
    no(ValueError, "activation", causal_conv, x, w, activation="gelu")
    no(ValueError, "initial_state must have shape", causal_conv, x, w, initial_state=i[:1])
    no(ValueError, "weight must be on", causal_conv, x, w.cpu())
    no(ValueError, "3 dimensions", causal_conv, x[0], w)
    no(ValueError, "one row of packed", causal_conv, x, w, cu_seqlens=[0, 10])
    no(ValueError, "rise from 0", causal_conv, x[:1], w, cu_seqlens=[0, 11])
    no(ValueError, "rise from 0", causal_conv, x[:1], w, cu_seqlens=[0, 7, 3, 10])
    no(TypeError, "int32 or int64", causal_conv, x[:1], w, cu_seqlens=torch.tensor([0.0, 10.0], device=dev))
    no(ValueError, "contiguous", causal_conv_step, x[:, 0], i.transpose(1, 2).contiguous().transpose(1, 2), w)
    no(TypeError, "int32 or int64", causal_conv_step, x[:, 0], i, w, slots=torch.zeros(2, device=dev))
    no(ValueError, "2 indices", causal_conv_step, x[:, 0], i, w, slots=torch.zeros(3, dtype=torch.int32, device=dev))
    no(TypeError, "A must be", selective_scan, **{**k, "A": k["A"].half()})
    no(ValueError, "1 to 128 states", selective_scan, **{**k, "A": torch.zeros(16, 129, device=dev)})
    no(ValueError, "groups dividing", selective_scan,
       **{**k, "B": k["B"].expand(2, 10, 3, 16), "C": k["C"].expand(2, 10, 3, 16)})
    no(ValueError, "C must have shape", selective_scan, **{**k, "C": k["C"][:, :5]})
    no(TypeError, "delta must be", selective_scan, **{**k, "delta": k["delta"].float()})
    no(ValueError, "z must have shape", selective_scan, **{**k, "z": k["z"][..., :8]})
    no(TypeError, "initial_state must be", selective_scan, **{**k, "initial_state": k["initial_state"].half()})
    one = {m: k[m][:, 0] for m in ("u", "delta", "B", "C", "z")}
    rest = {m: k[m] for m in ("A", "D", "delta_bias")}
    no(TypeError, "state must be", selective_scan_step, k["initial_state"].half(), **one, **rest)
    no(ValueError, "state must have shape", selective_scan_step, k["initial_state"][:1], **one, **rest)
    no(ValueError, "cannot require a gradient", selective_scan_step, k["initial_state"].requires_grad_(), **one, **rest)


@pytest.mark.gpu
def test_the_core_checks_its_arguments():
    """The C entries refuse what the Python layer would not send."""
    lib = _core.core_lib()
    from pto_einsum import _ops
    for name, packer in (("pe_causal_conv", ssm._CONV), ("pe_causal_conv_grad", ssm._CONV_GRAD),
                         ("pe_causal_conv_step", ssm._CONV_STEP), ("pe_selective_scan", ssm._SCAN),
                         ("pe_selective_scan_grad", ssm._SCAN_GRAD), ("pe_selective_scan_step", ssm._SCAN_STEP),
                         ("pe_group_norm", norm._NORM), ("pe_group_norm_grad", norm._NORM_GRAD)):
        fn = _ops.function(name)
        assert fn(b"\xff" * packer.size, None) == 1, name           # every field -1
        assert fn(None, None) == 1, name
        assert lib.pe_last_error() == 1
