"""The mixer layer (pto_einsum.mixer): contractions, convolution, scan and norm together,
against the same layer written with the float64 references; its tokens against its
prompts; a training step.

Tolerance for fp16: five contractions and three operators round their outputs to 11 bits,
each feeding the next with a gain near one: 8 x 2^-11, and the gate's product doubles it."""
import pytest
import torch

from pto_einsum import _core
from pto_einsum.mixer import SelectiveMixer
from pto_einsum.norm import group_norm_reference
from pto_einsum.ssm import causal_conv_reference, selective_scan_reference

TOL = {torch.float16: 16 * 2.0 ** -11, torch.float32: 1e-4}


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    assert a.shape == b.shape
    return ((a - b).norm() / b.norm()).item()


def reference(mix, h, p, cu=None):
    xz = torch.einsum("bte,ef->btf", h, p["w_in"])
    x, z = xz.chunk(2, -1)
    x = causal_conv_reference(x, p["conv_w"], p["conv_b"], activation="silu", cu_seqlens=cu)[0]
    r, B, C = mix._split(torch.einsum("btd,dr->btr", x, p["w_x"]))
    y, s = selective_scan_reference(x, torch.einsum("btr,rd->btd", r, p["w_dt"]), -torch.exp(p["A_log"]), B, C,
                                    p["D"], delta_bias=p["dt_bias"], delta_softplus=True, cu_seqlens=cu)
    y = group_norm_reference(y.flatten(0, 1), mix.heads, p["norm_w"], p["norm_b"], gate=z.flatten(0, 1))
    return torch.einsum("btd,de->bte", y.view(x.shape), p["w_out"]), s


def test_wrong_sizes_are_refused():
    with pytest.raises(ValueError, match="divide"):
        SelectiveMixer(32, 65, heads=2, device="cpu")
    with pytest.raises(TypeError, match="float16 or float32"):
        SelectiveMixer(32, 64, dtype=torch.bfloat16, device="cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
@pytest.mark.parametrize("B,T,cu", [(2, 48, None), (1, 64, [0, 10, 10, 64])])
def test_prompts_and_tokens(B, T, cu, dt):
    mix = SelectiveMixer(64, 128, heads=4, groups=2, dtype=dt, device="cuda", seed=1)
    g = torch.Generator().manual_seed(2)
    h = torch.randn(B, T, 64, generator=g).to(dt).cuda()
    n0 = _core.launch_count()
    y, state = mix(h, cu_seqlens=cu, return_state=True)
    assert _core.launch_count() - n0 >= 7
    r, s = reference(mix, h.double(), {k: v.double() for k, v in mix.params.items()}, cu)
    assert rel(y, r) <= TOL[dt] and rel(state["ssm"], s) <= TOL[dt]
    if cu is None:                                # the last tokens one by one
        _, part = mix(h[:, :T - 3].contiguous(), return_state=True)
        pool = mix.empty_state(7)
        slots = torch.tensor([6, 3], dtype=torch.int32, device="cuda")[:B]
        for k in pool:
            pool[k][slots.long()] = part[k]
        for t in range(T - 3, T):
            assert rel(mix.step(h[:, t].contiguous(), pool, slots), r[:, t]) <= TOL[dt]
        assert rel(pool["ssm"][slots.long()], s) <= TOL[dt]
    mix.cleanup()


@pytest.mark.gpu
def test_a_training_step():
    mix = SelectiveMixer(32, 64, heads=2, dtype=torch.float32, device="cuda", seed=3, requires_grad=True)
    g = torch.Generator().manual_seed(4)
    h = torch.randn(2, 24, 32, generator=g).cuda()
    target = torch.randn(2, 24, 32, generator=g).cuda()
    names = list(mix.params)

    def loss_of(y):
        return ((y - target.to(y.dtype)) ** 2).mean()

    loss = loss_of(mix(h))
    got = torch.autograd.grad(loss, [mix.params[n] for n in names])
    ref = {k: v.detach().double().requires_grad_() for k, v in mix.params.items()}
    want = torch.autograd.grad(loss_of(reference(mix, h.double(), ref)[0]), [ref[n] for n in names])
    for n, a, b in zip(names, got, want):
        assert rel(a, b) <= TOL[torch.float32], (n, rel(a, b))
    with torch.no_grad():
        for n, d in zip(names, got):
            mix.params[n] -= 0.05 * d
    assert loss_of(mix(h)) < loss
    mix.cleanup()
