"""Group norm (pto_einsum.norm) against its definition in float64: groups that stay in
registers and groups that do not, layouts, gradients, refusals.

Tolerances (relative 2-norm): outputs are rounded once (the type's unit roundoff u); the
statistics add up to n values in fp32 by trees and short runs, off by less than
sqrt(n) 2^-24 of the deviation, and each value passes a few more roundings: 2^-20 for
n up to 2^20. Where the mean is m deviations away, x - mean loses a factor m. Gradients
add the two means of products: four times that."""
import pytest
import torch

from pto_einsum import _core
from pto_einsum.norm import group_norm, group_norm_reference

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ROUND = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
FIXED = 2.0 ** -20


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    assert a.shape == b.shape
    if not b.numel():
        return 0.0
    off, size = (a - b).norm().item(), b.norm().item()
    return off / size if size else off


def rand(*shape, seed, dtype=F32, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).to(device)


CASES = [  # shape, groups
    ((1, 8), 1), ((5, 64), 4), ((300, 256), 8), ((7, 33), 3), ((64, 4096), 32), ((3, 8192), 1), ((2, 20000), 2),
    ((9, 16, 32), 4), ((2, 5, 7, 24), 3), ((2, 1024, 320), 32), ((1, 33, 31, 96), 1), ((3, 700, 50), 5),
    ((2, 9000, 8), 8), ((1, 5000, 7), 7), ((0, 16), 4), ((2, 0, 16), 4), ((1, 3, 260, 128), 2), ((4, 130), 130),
    ((70, 2722), 2), ((5, 24000), 2), ((3, 70000), 1), ((3, 40, 2600), 2), ((2, 31, 5000), 1)]


def inputs(shape, dt, seed=0):
    C = shape[-1]
    x = (rand(*shape, seed=seed + 1) * 1.5 + rand(C, seed=seed + 2)).to(dt)
    return x, rand(C, seed=seed + 3, dtype=dt), rand(C, seed=seed + 4, dtype=dt), rand(*shape, seed=seed + 5, dtype=dt)


def laid_out(x, layout):
    if layout == "columns":
        wide = torch.full((*x.shape[:-1], x.shape[-1] + 3), float("nan"), dtype=x.dtype, device=x.device)
        wide[..., 1:1 + x.shape[-1]] = x
        return wide[..., 1:1 + x.shape[-1]]
    return x


def test_host_tensors_and_wrong_arguments_are_refused():
    x = torch.zeros(4, 16)
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        group_norm(x, 4)
    with pytest.raises(ValueError, match="activation"):
        group_norm(x, 4, activation="relu")
    with pytest.raises(ValueError, match="exclude"):
        group_norm(x, 4, activation="silu", gate=x)
    with pytest.raises(ValueError, match="at least two"):
        group_norm(x[0], 4)


@pytest.mark.gpu
def test_refusals():
    x, w, b, z = inputs((4, 16), F16)

    def no(error, match, *a, **kw):
        with pytest.raises(error, match=match):
            group_norm(*a, **kw)

    no(ValueError, "groups must divide", x, 3)
    no(ValueError, "groups must divide", x, 0)
    no(TypeError, "weight must be", x, 4, w.float())
    no(ValueError, "bias must have shape", x, 4, w, b[:8])
    no(ValueError, "gate must have shape", x, 4, gate=z[:2])
    no(ValueError, "eps", x, 4, eps=-1.0)
    no(TypeError, "float32, float16", x.double(), 4)
    no(ValueError, "weight must be on", x, 4, w.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("layout", ["plain", "columns"])
@pytest.mark.parametrize("shape,groups", CASES)
def test_forward_and_gradients(shape, groups, layout, dt):
    x, w, b, z = inputs(shape, dt)
    dy = rand(*shape, seed=9, dtype=dt)
    # a channel of one value a group has no deviation: its xn and dx are zero over eps
    for act, gate, affine in (("silu", False, True), (None, True, True), (None, False, False)):
        leaves = [laid_out(x, layout)] + ([w, b] if affine else []) + ([laid_out(z, layout)] if gate else [])
        own = [t.detach().requires_grad_() for t in leaves]
        ref = [t.detach().double().requires_grad_() for t in leaves]

        def call(f, t):
            return f(t[0], groups, *(t[1:3] if affine else (None, None)), eps=1e-3, activation=act,
                     gate=t[-1] if gate else None)

        n0 = _core.launch_count()
        y, r = call(group_norm, own), call(group_norm_reference, ref)
        assert y.dtype == dt and y.is_contiguous() and y.shape == x.shape
        assert _core.launch_count() > n0 or not x.numel()
        assert rel(y, r) <= ROUND[dt] + FIXED, (act, gate)
        with torch.no_grad():
            assert torch.equal(y, call(group_norm, own))
        got = torch.autograd.grad(y, own, laid_out(dy, layout), retain_graph=True)
        want = torch.autograd.grad(r, ref, dy.double())
        for n, (g, h) in enumerate(zip(got, want)):
            assert g.dtype == dt and rel(g, h) <= 4 * (ROUND[dt] + FIXED) or h.norm() < 1e-9, (n, rel(g, h))
        again = torch.autograd.grad(y, own, laid_out(dy, layout))
        assert all(torch.equal(a, c) for a, c in zip(got, again))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("shape,groups", [
    ((640, 26000), 1), ((310, 26001), 1),                         # rows that share their sums' places in memory
    ((310, 8192), 1), ((700, 4104), 8),                           # and in shared memory
    ((40, 256, 1280), 32), ((8, 2100, 320), 32), ((2, 20000, 64), 4)])   # chunks in several waves
def test_many_rows_and_chunks(shape, groups, dt):
    test_forward_and_gradients(shape, groups, "plain", dt)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((40, 64), 4), ((2, 3000, 64), 4)])
def test_gradients_against_differences(shape, groups):
    x, w, b, z = inputs(shape, F32)
    t = [x, w, b, z]
    dy = rand(*shape, seed=11)
    own = [v.detach().requires_grad_() for v in t]
    got = torch.autograd.grad(group_norm(own[0], groups, own[1], own[2], gate=own[3]), own, dy)
    eps = 1e-5
    for i in range(4):
        v = rand(*t[i].shape, seed=20 + i).double()
        f = []
        for s in (1, -1):
            a = [u.double() for u in t]
            a[i] = a[i] + s * eps * v
            f.append((group_norm_reference(a[0], groups, a[1], a[2], gate=a[3]) * dy).sum().item())
        want, have = (f[0] - f[1]) / (2 * eps), (got[i].double() * v).sum().item()
        size = (got[i].double() * v).norm().item()
        assert abs(want - have) <= 1e-6 * abs(want) + 40 * FIXED * size, (i, want, have)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((16, 512), 4), ((2, 4000, 64), 4)])
def test_a_mean_far_from_zero(shape, groups):
    """1000 deviations away: a difference of squares would keep nothing of the variance."""
    x = rand(*shape, seed=1) + 1000.0
    assert rel(group_norm(x, groups), group_norm_reference(x, groups)) <= 1000 * 2.0 ** -24 + FIXED


@pytest.mark.gpu
def test_constant_rows_and_infinities():
    x = rand(6, 64, seed=1)
    x[2] = 5.0
    y = group_norm(x, 4)
    assert (y[2] == 0).all()                     # no deviation: zero over the root of eps
    x2 = x.clone()
    x2[4, 20] = float("inf")
    y2 = group_norm(x2, 4)
    assert torch.isnan(y2[4, 16:32]).any()
    keep = torch.ones(6, 64, dtype=torch.bool, device="cuda")
    keep[4, 16:32] = False
    assert torch.equal(y2[keep], y[keep])
