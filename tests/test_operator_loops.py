"""The recurrent-mixer operators at sizes where a thread takes many tokens, rows or requests: the steady
state of their loops, which small sizes do not enter. Against the float64 definitions.

Tolerances (relative 2-norm) as at the small sizes: an output has its type's unit roundoff u and
2^-20 of the arithmetic; gradients add products of two such quantities, four times that. A
scan's error grows with the root of the tokens that a state remembers, 2^-21 each and a factor of
eight for their spread."""
import pytest
import torch

from pto_einsum import _core
from pto_einsum.norm import group_norm, group_norm_reference
from pto_einsum.ssm import (causal_conv, causal_conv_reference, selective_scan, selective_scan_reference,
                            selective_scan_step)

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ROUND = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
STEP, FIXED = 2.0 ** -21, 2.0 ** -20
TYPES = [F32, F16, BF16]


def rand(*shape, seed, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    assert a.shape == b.shape and torch.isfinite(a).all()
    return ((a - b).norm() / b.norm()).item()


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def vector(dt, layout):
    """Elements a load."""
    return 1 if layout == "columns" else 4 if dt == F32 else 8


def laid_out(x, layout):
    if layout == "columns":                      # a slice of wider rows, off the 16-byte boundary
        wide = torch.full((*x.shape[:-1], x.shape[-1] + 5), float("nan"), dtype=x.dtype, device=x.device)
        wide[..., 3:3 + x.shape[-1]] = x
        return wide[..., 3:3 + x.shape[-1]]
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("layout", ["plain", "columns"])
@pytest.mark.parametrize("B,T,C,W,cu", [(1, 6000, 2048, 4, [0, 0, 1, 3, 1000, 1007, 2500, 2500, 2533, 4999, 6000]),
                                        (3, 2011, 2048, 2, None), (2, 3001, 2048, 3, None)])
def test_convolution_walks(B, T, C, W, cu, layout, dt):
    # forward two blocks of 256 threads an SM (backward one or two): a thread walks more tokens
    # than its queue of eight has slots, twice over and with a remainder
    assert B * T * C // vector(dt, layout) > 16 * 2 * 256 * sms()
    n = len(cu) - 1 if cu else B
    x, w = laid_out(rand(B, T, C, seed=1, dtype=dt), layout), rand(C, W, seed=2, dtype=dt) * W ** -0.5
    t = [x, w.to(dt), rand(C, seed=3, dtype=dt), rand(n, W - 1, C, seed=4, dtype=dt)]
    dy, dend = laid_out(rand(B, T, C, seed=5, dtype=dt), layout), rand(n, W - 1, C, seed=6, dtype=dt)
    own = [v.detach().requires_grad_() for v in t]
    ref = [v.detach().double().requires_grad_() for v in t]
    for act in ("silu", None):
        y, end = causal_conv(*own[:3], activation=act, initial_state=own[3], cu_seqlens=cu, return_state=True)
        r, rend = causal_conv_reference(*ref[:3], activation=act, initial_state=ref[3], cu_seqlens=cu)
        assert rel(y, r) <= ROUND[dt] + FIXED and torch.equal(end.double(), rend)
        got = torch.autograd.grad([y, end], own, [dy, dend])
        want = torch.autograd.grad([r, rend], ref, [dy.double(), dend.double()])
        for name, a, b in zip(("x", "weight", "bias", "initial_state"), got, want):
            assert a.dtype == dt and rel(a, b) <= 4 * (ROUND[dt] + FIXED), (name, rel(a, b))
    assert _core.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("N", [16, 15])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_two_requests_a_thread(index, N, dt):
    """An odd last request, and skipped ones beside ones that are not."""
    B, D, G, pool = 257, 4096, 2, 300
    assert D // 64 * B >= 32 * sms()
    u, delta, z = (rand(B, D, seed=s, dtype=dt) for s in (1, 2, 3))
    Bm, C = rand(B, G, N, seed=4, dtype=dt), rand(B, G, N, seed=5, dtype=dt)
    A, skip, bias = -torch.exp(rand(D, N, seed=6)), rand(D, seed=7), rand(D, seed=8) - 2
    state = rand(pool, D, N, seed=9)
    slots = torch.randperm(pool, generator=torch.Generator().manual_seed(10))[:B]
    slots[[0, 17, 100, 101, 254]] = -1
    on, before = (slots >= 0).cuda(), state.clone()
    at = slots[slots >= 0].cuda()
    y = selective_scan_step(state, u, delta, A, Bm, C, skip, z=z, delta_bias=bias, delta_softplus=True,
                            slots=slots.to(index).cuda())
    one = [t[on][:, None] for t in (u, delta, Bm, C, z)]
    r, end = selective_scan_reference(one[0], one[1], A, one[2], one[3], skip, z=one[4], delta_bias=bias,
                                      delta_softplus=True, initial_state=before[at])
    assert rel(y[on], r[:, 0]) <= ROUND[dt] + FIXED + STEP and rel(state[at], end) <= FIXED + STEP
    assert (y[~on] == 0).all()
    rest = torch.ones(pool, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert torch.equal(state[rest], before[rest]) and _core.device_error() == 0


ROWS = [  # shape, groups: rows of several rounds a group of lanes
    ((3000, 4096), 32), ((2000, 4096), 8),       # part of a warp a group, one load a lane and two
    ((700, 2048), 1), ((700, 4096), 1),          # a block a group
    ((3000, 1608), 8), ((3000, 808), 8),         # eight and four single elements a lane
    ((3000, 9, 64), 4), ((2500, 12, 64), 1)]     # several places


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("layout", ["plain", "columns"])
@pytest.mark.parametrize("shape,groups", ROWS)
def test_norm_of_many_rows(shape, groups, layout, dt):
    C = shape[-1]
    x = laid_out((rand(*shape, seed=1) * 1.5 + rand(C, seed=2)).to(dt), layout)
    z, dy = laid_out(rand(*shape, seed=5, dtype=dt), layout), laid_out(rand(*shape, seed=6, dtype=dt), layout)
    w, b = rand(C, seed=3, dtype=dt), rand(C, seed=4, dtype=dt)
    for act, leaves in (("silu", [x, w, b]), (None, [x, w, b, z]), (None, [x])):
        own = [t.detach().requires_grad_() for t in leaves]
        ref = [t.detach().double().requires_grad_() for t in leaves]

        def call(f, t):
            return f(t[0], groups, *t[1:3], activation=act, gate=t[3] if len(t) > 3 else None)

        n0 = _core.launch_count()
        y, r = call(group_norm, own), call(group_norm_reference, ref)
        assert y.dtype == dt and rel(y, r) <= ROUND[dt] + FIXED
        if layout == "plain":
            assert _core.launch_count() == n0 + 1        # in registers, one pass
        got, want = torch.autograd.grad(y, own, dy), torch.autograd.grad(r, ref, dy.double())
        for g, h in zip(got, want):
            assert g.dtype == dt and rel(g, h) <= 4 * (ROUND[dt] + FIXED), rel(g, h)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", [(4, 130), (300, 7), (2, 40, 24)])
def test_groups_of_one_value(shape, dt):
    """One value a group and place: with a single place no deviation, so that xn, dx and the filter's
    gradient are zero but for roundings; several types of results that a relative bound cannot see."""
    C = shape[-1]
    x, w, b, dy = (rand(*s, seed=i, dtype=dt) for i, s in enumerate((shape, (C,), (C,), shape)))
    own = [t.detach().requires_grad_() for t in (x, w, b)]
    y = group_norm(own[0], C, own[1], own[2], eps=1e-3)
    got = torch.autograd.grad(y, own, dy)
    ref = [t.detach().double().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(group_norm_reference(ref[0], C, ref[1], ref[2], eps=1e-3), ref, dy.double())
    # sizes of the terms that cancel: dout w rstd in dx, the sum of dout xn in the filter's gradient
    rows = dy.double().flatten(0, -2).abs().sum(0).max().item()
    size = [(dy * w).abs().max().item() * 1e-3 ** -0.5, rows, rows]
    for g, h, s in zip(got, want, size):
        assert g.dtype == dt and torch.isfinite(g).all()
        assert (g.double() - h).abs().max().item() <= 4 * (ROUND[dt] * h.abs().max().item() + FIXED * s)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("layout", ["plain", "columns"])
@pytest.mark.parametrize("T,D,N,G,cu", [(3000, 48, 16, 2, None), (2600, 24, 5, 1, [0, 1200, 1200, 1300, 2600])])
def test_scans_split_along_time(T, D, N, G, cu, layout, dt):
    n = len(cu) - 1 if cu else 1
    act = {m: laid_out(rand(*s, seed=i, dtype=dt), layout) for i, (m, s) in enumerate(
        dict(u=(1, T, D), delta=(1, T, D), B=(1, T, G, N), C=(1, T, G, N), z=(1, T, D)).items())}
    k = dict(act, A=-torch.exp(rand(D, N, seed=10)), D=rand(D, seed=11), delta_bias=rand(D, seed=12) - 4,
             initial_state=rand(n, D, N, seed=13))
    dy, dend = laid_out(rand(1, T, D, seed=14, dtype=dt), layout), rand(n, D, N, seed=15)
    own = {m: t.detach().requires_grad_() for m, t in k.items()}
    ref = {m: t.detach().double().requires_grad_() for m, t in k.items()}
    tol = FIXED + T ** 0.5 * 8 * STEP
    n0 = _core.launch_count()
    y, end = selective_scan(**own, delta_softplus=True, cu_seqlens=cu, return_state=True)
    assert _core.launch_count() == n0 + 3                 # states of the pieces, their joining, the scan
    r, rend = selective_scan_reference(**ref, delta_softplus=True, cu_seqlens=cu)
    assert rel(y, r) <= ROUND[dt] + tol and rel(end, rend) <= tol
    n0 = _core.launch_count()
    got = torch.autograd.grad([y, end], list(own.values()), [dy, dend])
    assert _core.launch_count() == n0 + 5                 # the same backwards, and two launches of sums
    want = torch.autograd.grad([r, rend], list(ref.values()), [dy.double(), dend.double()])
    for m, a, b in zip(k, got, want):
        assert a.dtype == k[m].dtype and rel(a, b) <= 4 * (ROUND[k[m].dtype] + tol), (m, rel(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16])
@pytest.mark.parametrize("nseq", [64, 128, 129, 300])
def test_many_packed_sequences(nseq, dt):
    """Around the number of sequences up to which the longest go first; a sixth of them empty."""
    T, D, N = 1500, 200, 16
    g = torch.Generator().manual_seed(nseq)
    cuts = torch.randint(0, T + 1, (nseq - 1,), generator=g)
    again = torch.randint(0, nseq - 1, (nseq // 6,), generator=g)
    cuts[again] = cuts[(again + 1) % (nseq - 1)]
    cu = [0, *cuts.sort().values.tolist(), T]
    k = {m: rand(*s, seed=i, dtype=dt) for i, (m, s) in enumerate(
        dict(u=(1, T, D), delta=(1, T, D), B=(1, T, 1, N), C=(1, T, 1, N), z=(1, T, D)).items())}
    k.update(A=-torch.exp(rand(D, N, seed=10)), D=rand(D, seed=11), delta_bias=rand(D, seed=12) - 4,
             initial_state=rand(nseq, D, N, seed=13))
    dy, dend = rand(1, T, D, seed=14, dtype=dt), rand(nseq, D, N, seed=15)
    own = {m: t.detach().requires_grad_() for m, t in k.items()}
    ref = {m: t.detach().double().requires_grad_() for m, t in k.items()}
    tol = FIXED + T ** 0.5 * 8 * STEP
    table = torch.tensor(cu, dtype=torch.int32, device="cuda")
    y, end = selective_scan(**own, delta_softplus=True, cu_seqlens=table, return_state=True)
    r, rend = selective_scan_reference(**ref, delta_softplus=True, cu_seqlens=cu)
    assert rel(y, r) <= ROUND[dt] + tol and rel(end, rend) <= tol
    got = torch.autograd.grad([y, end], list(own.values()), [dy, dend])
    want = torch.autograd.grad([r, rend], list(ref.values()), [dy.double(), dend.double()])
    for m, a, b in zip(k, got, want):
        assert a.dtype == k[m].dtype and rel(a, b) <= 4 * (ROUND[k[m].dtype] + tol), (m, rel(a, b))
    x, w, b = k["u"], rand(D, 4, seed=20, dtype=dt), rand(D, seed=21, dtype=dt)
    y, end = causal_conv(x, w, b, activation="silu", cu_seqlens=table, return_state=True)
    r, rend = causal_conv_reference(x, w, b, activation="silu", cu_seqlens=cu)
    assert rel(y, r) <= ROUND[dt] + FIXED and torch.equal(end.double(), rend)
    assert _core.device_error() == 0
