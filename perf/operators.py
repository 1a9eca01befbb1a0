"""Cases of the recurrent-mixer operators: the short causal convolution, the selective state space
scan, their single-token forms and the channels-last group norm, each in a plain form (elementary
torch operations in 32 bits) and as the calls a user makes of this library.

listed() and draw() name cases, prepare() makes what a program holds before the call, run() is one
pass, work() the bytes and operations the pass cannot do without, exact() the answer in 64 bits.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- cases --------------------------------------------------------------------------------------
# "nseq" 0: a batch of B sequences of T tokens. nseq > 0: B = 1 and T tokens of nseq sequences of
# different lengths, packed end to end ("cu_seqlens"), an empty one among them from nseq = 3 on.
def listed():
    return [
        # prompts of many requests packed into one call of a serving engine, carrying each request's
        # convolution state: inner channels plus the scan's B and C columns
        dict(name="conv prompts packed", op="conv", B=1, T=16384, nseq=24, C=4352, W=4, dtype="bf16", bias=True,
             silu=True, state=True, grad=False),
        # one layer's training step on its convolution
        dict(name="conv training", op="conv", B=4, T=2048, nseq=0, C=2048, W=4, dtype="f16", bias=True, silu=True,
             state=False, grad=True),
        # one token of one request: the latency of a decode step
        dict(name="conv token", op="conv_step", B=1, C=2048, W=4, dtype="bf16", bias=True, silu=True, slots=0),
        # one token of each request of a large decode batch, states held in a pool of slots
        dict(name="conv tokens in slots", op="conv_step", B=512, C=4352, W=4, dtype="f16", bias=True, silu=True,
             slots=640),
        # one long prompt: few channels, a long time axis
        dict(name="scan long prompt", op="scan", B=1, T=32768, nseq=0, D=2048, N=16, G=1, dtype="bf16", gate=True,
             skip=True, state=False, grad=False),
        # packed prompts that go on from earlier states
        dict(name="scan prompts packed", op="scan", B=1, T=8192, nseq=17, D=4096, N=16, G=1, dtype="f16", gate=True,
             skip=True, state=True, grad=False),
        # one layer's training step on its scan
        dict(name="scan training", op="scan", B=4, T=2048, nseq=0, D=2048, N=16, G=1, dtype="bf16", gate=True,
             skip=True, state=False, grad=True),
        # the same in 32 bits with odd sizes, three groups of B and C, and a gradient of the first state
        dict(name="scan training odd", op="scan", B=3, T=509, nseq=0, D=390, N=24, G=3, dtype="f32", gate=False,
             skip=True, state=True, grad=True),
        # one token of one request
        dict(name="scan token", op="scan_step", B=1, D=2048, N=16, G=1, dtype="bf16", gate=True, skip=True, slots=0),
        # one token of each request of a large decode batch
        dict(name="scan tokens in slots", op="scan_step", B=256, D=4096, N=16, G=1, dtype="f16", gate=True, skip=True,
             slots=320),
        # the gated norm over head groups after a recurrent mixer, one row a token, in training
        dict(name="norm training", op="norm", N=8192, S=1, C=4096, G=32, dtype="bf16", affine=True, act="gate",
             grad=True),
        # a feature map, channels last: statistics over 64 x 64 places and ten channels a group
        dict(name="norm map", op="norm", N=4, S=4096, C=320, G=32, dtype="f16", affine=True, act="silu", grad=False),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _channels(rng, lo, hi, groups=1):
    """A usual width, or any with an odd number of channels a group."""
    if rng.random() < 0.6:
        return rng.choice([c for c in (64, 96, 128, 192, 256, 320, 384, 512, 640, 768, 1024, 1280, 1536, 2048, 2560,
                                       4096, 5120, 8192) if lo <= c <= hi and c % groups == 0])
    return max(1, _between(rng, lo, hi - groups) // groups // 2 * 2 - 1) * groups


def _cost(case):
    w = work(case)
    return w["bytes"] + w["flops"] / 10


def draw(rng):
    most = max(map(_cost, listed()))
    while True:
        case = _draw(rng)
        if _cost(case) <= most:
            return case


def _draw(rng):
    op = rng.choice(["conv", "conv", "conv_step", "scan", "scan", "scan_step", "norm", "norm"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "conv":
        grad = rng.random() < 0.5
        C = _channels(rng, 64, 8192)
        T = _between(rng, 1, min(32768, (16 << 20 if grad else 64 << 20) // C))
        packed = rng.random() < 0.5
        B = 1 if packed else max(1, min(16, _between(rng, 1, 16)) if T < 4096 else 1)
        T = max(1, T // B)
        return dict(op=op, B=B, T=T, nseq=rng.randint(1, 32) if packed else 0, C=C, W=rng.choice([2, 3, 4, 4, 4]),
                    dtype=dtype, bias=rng.random() < 0.7, silu=rng.random() < 0.7, state=rng.random() < 0.5, grad=grad)
    if op == "conv_step":
        B = _between(rng, 1, 512)
        return dict(op=op, B=B, C=_channels(rng, 64, 4352), W=rng.choice([2, 3, 4, 4, 4]), dtype=dtype,
                    bias=rng.random() < 0.7, silu=rng.random() < 0.7, slots=rng.choice([0, B + rng.randint(1, 128)]))
    if op == "scan":
        grad = rng.random() < 0.5
        G = rng.choice([1, 1, 1, 2, 4])
        N = rng.choice([4, 8, 16, 16, 16, 16, 32, 64, rng.randint(1, 64)])
        D = _channels(rng, 64, 4096, G)
        T = _between(rng, 1, max(2, min(32768, (256 << 20 if grad else 1 << 30) // (D * N))))
        packed = rng.random() < 0.4
        B = 1 if packed else max(1, _between(rng, 1, 8) if T < 4096 else 1)
        T = max(1, T // B)
        return dict(op=op, B=B, T=T, nseq=rng.randint(1, 32) if packed else 0, D=D, N=N, G=G, dtype=dtype,
                    gate=rng.random() < 0.7, skip=rng.random() < 0.8, state=rng.random() < 0.5, grad=grad)
    if op == "scan_step":
        B, G = _between(rng, 1, 256), rng.choice([1, 1, 2])
        return dict(op=op, B=B, D=_channels(rng, 64, 4096, G),
                    N=rng.choice([8, 16, 16, 16, 32, rng.randint(1, 32)]), G=G, dtype=dtype, gate=rng.random() < 0.7,
                    skip=rng.random() < 0.8, slots=rng.choice([0, B + rng.randint(1, 64)]))
    G = rng.choice([1, 2, 8, 16, 32, 32])
    C = _channels(rng, 64, 4096, G)
    cells = (32 << 20) // C
    tokens = rng.random() < 0.5
    S = 1 if tokens else _between(rng, 2, min(16384, cells))
    N = _between(rng, 1, max(2, min(16384 if tokens else 64, cells // S)))
    return dict(op=op, N=N, S=S, C=C, G=G, dtype=dtype, affine=rng.random() < 0.8,
                act=rng.choice(["none", "silu", "gate"]), grad=rng.random() < 0.5)


# ---- what a program has in hand -----------------------------------------------------------------
def _lengths(case, seed):
    """Cumulative lengths of the packed sequences: random cuts, the second sequence empty from three on."""
    import random
    rng = random.Random(seed * 7919 + case["T"])
    cuts = sorted(rng.randint(0, case["T"]) for _ in range(case["nseq"] - 1))
    if case["nseq"] >= 3:
        cuts[1] = cuts[0]
    return [0] + cuts + [case["T"]]


def _makers(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    def slots(n, pool):
        return torch.randperm(pool, generator=g, device="cuda")[:n].to(torch.int32)

    return normal, uniform, slots


def _bounds(case, seed):
    if not case["nseq"]:
        return case["B"], None
    return case["nseq"], torch.tensor(_lengths(case, seed), dtype=torch.int32, device="cuda")


def _scan_weights(case, normal, uniform):
    """A, D and the bias of delta as they are set before training and stay close to after it: decays of 1 to N
    a unit of delta, step sizes of 0.001 to 0.1."""
    D, N = case["D"], case["N"]
    A = -torch.arange(1, N + 1, device="cuda").float() * torch.exp(normal(D, N, scale=0.1))
    dt = torch.exp(uniform(D) * math.log(100.0)) * 1e-3
    return A, normal(D, scale=0.1) + 1.0 if case["skip"] else None, dt + torch.log(-torch.expm1(-dt))


def prepare(case, seed):
    normal, uniform, slots = _makers(seed)
    op, dt = case["op"], TYPES[case["dtype"]]
    s = dict(case=case)
    if op in ("conv", "conv_step"):
        C, W = case["C"], case["W"]
        s["w"] = normal(C, W, dtype=dt, scale=W ** -0.5)
        s["b"] = normal(C, dtype=dt, scale=0.1) if case["bias"] else None
    if op == "conv":
        nseq, s["cu"] = _bounds(case, seed)
        s["x"] = normal(case["B"], case["T"], 2 * C, dtype=dt)[..., :C]  # one half of a projection's columns
        s["init"] = normal(nseq, W - 1, C, dtype=dt) if case["state"] else None
        if case["grad"]:
            s["dout"] = normal(case["B"], case["T"], C, dtype=dt)
            s["x"] = s["x"].detach()
            s["wrt"] = [k for k in ("x", "w", "b", "init") if s[k] is not None]
    elif op == "conv_step":
        s["x"] = normal(case["B"], 2 * C, dtype=dt)[:, :C]
        s["state"] = normal(case["slots"] or case["B"], W - 1, C, dtype=dt)
        s["slots"] = slots(case["B"], case["slots"]) if case["slots"] else None
    elif op == "scan":
        nseq, s["cu"] = _bounds(case, seed)
        B, T, D, N, G = (case[k] for k in "BTDNG")
        s["u"] = normal(B, T, D, dtype=dt)
        s["delta"] = normal(B, T, D, dtype=dt)
        cols = normal(B, T, 2, G, N, dtype=dt)  # B and C are columns of one projection
        s["Bm"], s["Cm"] = cols[:, :, 0], cols[:, :, 1]
        s["z"] = normal(B, T, 2 * D, dtype=dt)[..., D:] if case["gate"] else None
        s["A"], s["D"], s["bias"] = _scan_weights(case, normal, uniform)
        s["init"] = normal(nseq, D, N) if case["state"] else None
        if case["grad"]:
            s["dout"] = normal(B, T, D, dtype=dt)
            for k in ("Bm", "Cm", "z"):
                s[k] = s[k].detach() if s[k] is not None else None
            s["wrt"] = [k for k in ("u", "delta", "A", "Bm", "Cm", "D", "z", "bias", "init") if s[k] is not None]
    elif op == "scan_step":
        B, D, N, G = (case[k] for k in "BDNG")
        s["u"], s["delta"] = normal(B, D, dtype=dt), normal(B, D, dtype=dt)
        cols = normal(B, 2, G, N, dtype=dt)
        s["Bm"], s["Cm"] = cols[:, 0], cols[:, 1]
        s["z"] = normal(B, 2 * D, dtype=dt)[:, D:] if case["gate"] else None
        s["A"], s["D"], s["bias"] = _scan_weights(case, normal, uniform)
        s["state"] = normal(case["slots"] or B, D, N)
        s["slots"] = slots(B, case["slots"]) if case["slots"] else None
    else:
        shape = (case["N"], case["C"]) if case["S"] == 1 else (case["N"], case["S"], case["C"])
        s["x"] = (normal(*shape) * 1.5 + normal(case["C"]) * 0.5).to(dt)
        s["w"] = normal(case["C"], dtype=dt, scale=0.2) + 1 if case["affine"] else None
        s["b"] = normal(case["C"], dtype=dt, scale=0.2) if case["affine"] else None
        s["z"] = normal(*shape, dtype=dt) if case["act"] == "gate" else None
        if case["grad"]:
            s["dout"] = normal(*shape, dtype=dt)
            s["wrt"] = [k for k in ("x", "w", "b", "z") if s[k] is not None]
    for k in s.get("wrt", ()):
        s[k].requires_grad_(True)
    return s


# ---- one pass -----------------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return PLAIN[s["case"]["op"]](s, s["case"])


def _run_own(s):
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pto-einsum_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from pto_einsum.norm import group_norm
    from pto_einsum.ssm import causal_conv, causal_conv_step, selective_scan, selective_scan_step
    c = s["case"]
    act = "silu" if c.get("silu") else None
    if c["op"] == "conv":
        r = causal_conv(s["x"], s["w"], s["b"], activation=act, initial_state=s["init"], cu_seqlens=s["cu"],
                        return_state=not c["grad"])
    elif c["op"] == "conv_step":
        y = causal_conv_step(s["x"], s["state"], s["w"], s["b"], activation=act, slots=s["slots"])
        return {"out": y, "state": s["state"]}
    elif c["op"] == "scan":
        r = selective_scan(s["u"], s["delta"], s["A"], s["Bm"], s["Cm"], s["D"], z=s["z"], delta_bias=s["bias"],
                           delta_softplus=True, initial_state=s["init"], cu_seqlens=s["cu"],
                           return_state=not c["grad"])
    elif c["op"] == "scan_step":
        y = selective_scan_step(s["state"], s["u"], s["delta"], s["A"], s["Bm"], s["Cm"], s["D"], z=s["z"],
                                delta_bias=s["bias"], delta_softplus=True, slots=s["slots"])
        return {"out": y, "state": s["state"]}
    else:
        r = group_norm(s["x"], c["G"], s["w"], s["b"], activation="silu" if c["act"] == "silu" else None,
                       gate=s["z"], eps=1e-5)
    if c["grad"]:
        return {"out": r.detach(), "grad": list(torch.autograd.grad(r, [s[k] for k in s["wrt"]], s["dout"]))}
    return {"out": r} if c["op"] == "norm" else {"out": r[0], "state": r[1]}


# ---- plain forms --------------------------------------------------------------------------------
def _f(x):
    return None if x is None else x.float()


def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _softplus(x):
    return x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))


def _sequences(s, c):
    """For the tokens of all sequences in one row: each token's sequence, and the sequences' bounds."""
    T = c["B"] * c["T"]
    cu = torch.arange(c["B"] + 1, device="cuda") * c["T"] if s["cu"] is None else s["cu"].long()
    return torch.bucketize(torch.arange(T, device="cuda"), cu[1:], right=True), cu


def _conv(s, c):
    W, C = c["W"], c["C"]
    seq, cu = _sequences(s, c)
    T, S = seq.numel(), cu.numel() - 1
    x, w, b, init = _f(s["x"]).reshape(T, C), _f(s["w"]), _f(s["b"]), _f(s["init"])
    # all sequences in one row, W - 1 earlier inputs before each
    place = torch.arange(T, device="cuda") + (W - 1) * (seq + 1)
    before = (cu[:-1] + (W - 1) * torch.arange(S, device="cuda"))[:, None] + torch.arange(W - 1, device="cuda")
    row = x.new_zeros(T + S * (W - 1), C)
    row[place] = x
    if init is not None:
        row[before] = init
    win = row.unfold(0, W, 1)[place - (W - 1)]  # [T, C, W]
    p = (win * w).sum(-1)
    p = p + b if b is not None else p
    y = p * _sigmoid(p) if c["silu"] else p
    out = y.to(s["x"].dtype).reshape(s["x"].shape)
    if not c["grad"]:
        return {"out": out, "state": row[before + (cu[1:] - cu[:-1])[:, None]].to(s["x"].dtype)}
    g = _f(s["dout"]).reshape(T, C)
    if c["silu"]:
        q = _sigmoid(p)
        g = g * q * (1 + p * (1 - q))
    grow = x.new_zeros(T + S * (W - 1) + W - 1, C)
    grow[place] = g
    drow = (grow.unfold(0, W, 1) * w.flip(-1)).sum(-1)
    d = {"x": drow[place].reshape(s["x"].shape), "w": (win * g[..., None]).sum(0), "b": g.sum(0), "init": drow[before]}
    return {"out": out, "grad": [d[k].to(s[k].dtype) for k in s["wrt"]]}


def _conv_step(s, c):
    idx = slice(None) if s["slots"] is None else s["slots"].long()
    win = torch.cat([s["state"][idx], s["x"][:, None]], 1)  # [B, W, C]
    p = (_f(win) * _f(s["w"]).t()).sum(1)
    p = p + _f(s["b"]) if s["b"] is not None else p
    y = p * _sigmoid(p) if c["silu"] else p
    s["state"][idx] = win[:, 1:]
    return {"out": y.to(s["x"].dtype), "state": s["state"]}


def _recur(a, b):
    """h[t] = a[t] h[t-1] + b[t] along the first axis by doubling: after the pass with distance k, row t holds the
    composition of the last 2k steps. One loop of log2(T) passes over whole tensors."""
    k = 1
    while k < a.shape[0]:
        b = torch.cat([b[:k], b[k:] + a[k:] * b[:-k]])
        a = torch.cat([a[:k], a[k:] * a[:-k]])
        k *= 2
    return b


def _heads(m, c, T):
    """B or C of each channel's group: [T, D, N]."""
    return _f(m).reshape(T, c["G"], 1, c["N"]).expand(T, c["G"], c["D"] // c["G"], c["N"]).reshape(T, c["D"], c["N"])


def _scan(s, c):
    D, N, G = c["D"], c["N"], c["G"]
    seq, cu = _sequences(s, c)
    T, S = seq.numel(), cu.numel() - 1
    u, raw, A, z = _f(s["u"]).reshape(T, D), _f(s["delta"]).reshape(T, D) + s["bias"], s["A"], _f(s["z"])
    dt = _softplus(raw)
    Bm, Cm = _heads(s["Bm"], c, T), _heads(s["Cm"], c, T)
    h0 = A.new_zeros(S, D, N) if s["init"] is None else s["init"]
    some = cu[1:] > cu[:-1]
    first, last = cu[:-1].clamp(max=T - 1), (cu[1:] - 1).clamp(min=0)
    starts = torch.zeros(T, device="cuda").index_add_(0, first, some.float())[:, None, None]
    a = torch.exp(dt[..., None] * A)
    h_in = h0[seq] * starts  # what each sequence starts from, at its first token
    h = _recur(a * (1 - starts), (dt * u)[..., None] * Bm + a * h_in)
    y = (Cm * h).sum(-1)
    y = y + s["D"] * u if s["D"] is not None else y
    zz = z.reshape(T, D) if z is not None else None
    out = y * zz * _sigmoid(zz) if z is not None else y
    out = out.to(s["u"].dtype).reshape(s["u"].shape)
    if not c["grad"]:
        return {"out": out, "state": torch.where(some[:, None, None], h[last], h0)}
    dy, d = _f(s["dout"]).reshape(T, D), {}
    if z is not None:
        q = _sigmoid(zz)
        d["z"] = dy * y * q * (1 + zz * (1 - q))
        dy = dy * zz * q
    back = torch.cat([(a * (1 - starts))[1:], torch.zeros_like(a[:1])])  # a[t+1] within the sequence
    g = _recur(back.flip(0), (Cm * dy[..., None]).flip(0)).flip(0)
    hp = torch.cat([torch.zeros_like(h[:1]), h[:-1]]) * (1 - starts) + h_in
    e = g * hp * a
    gB = (g * Bm).sum(-1)
    ddt = gB * u + (e * A).sum(-1)
    group = lambda m: m.reshape(T, G, D // G, N).sum(2)  # noqa: E731
    d["u"] = gB * dt + (dy * s["D"] if s["D"] is not None else 0)
    d["A"], d["D"] = (e * dt[..., None]).sum(0), (dy * u).sum(0)
    d["Bm"], d["Cm"] = group(g * (dt * u)[..., None]), group(h * dy[..., None])
    d["delta"] = ddt * _sigmoid(raw)
    d["bias"] = d["delta"].sum(0)
    d["init"] = (a * g)[first] * some[:, None, None]
    return {"out": out, "grad": [d[k].reshape(s[k].shape).to(s[k].dtype) for k in s["wrt"]]}


def _scan_step(s, c):
    idx = slice(None) if s["slots"] is None else s["slots"].long()
    n = s["u"].shape[0]
    u, dt = _f(s["u"]), _softplus(_f(s["delta"]) + s["bias"])
    h = torch.exp(dt[..., None] * s["A"]) * s["state"][idx] + (dt * u)[..., None] * _heads(s["Bm"], c, n)
    y = (_heads(s["Cm"], c, n) * h).sum(-1)
    y = y + s["D"] * u if s["D"] is not None else y
    y = y * _f(s["z"]) * _sigmoid(_f(s["z"])) if s["z"] is not None else y
    s["state"][idx] = h
    return {"out": y.to(s["u"].dtype), "state": s["state"]}


def _norm(s, c):
    N, S, C, G = (c[k] for k in "NSCG")
    x = _f(s["x"]).reshape(N, S, G, C // G)
    w, b, z = (_f(s[k]) for k in ("w", "b", "z"))
    xc = x - x.mean((1, 3), keepdim=True)
    r = torch.rsqrt((xc * xc).mean((1, 3), keepdim=True) + 1e-5)
    xn = xc * r
    v = xn.reshape(N, S, C)
    v = v * w + b if w is not None else v
    p = z.reshape(N, S, C) if z is not None else v
    q = _sigmoid(p)
    y = v if c["act"] == "none" else v * p * q if z is not None else v * q
    out = y.to(s["x"].dtype).reshape(s["x"].shape)
    if not c["grad"]:
        return {"out": out}
    g, d = _f(s["dout"]).reshape(N, S, C), {}
    slope = q * (1 + p * (1 - q))
    if z is not None:
        d["z"], g = g * v * slope, g * p * q
    elif c["act"] == "silu":
        g = g * slope
    d["w"], d["b"] = (g * xn.reshape(N, S, C)).sum((0, 1)), g.sum((0, 1))
    gx = (g * w if w is not None else g).reshape(N, S, G, C // G)
    d["x"] = r * (gx - gx.mean((1, 3), keepdim=True) - xn * (gx * xn).mean((1, 3), keepdim=True))
    return {"out": out, "grad": [d[k].reshape(s[k].shape).to(s[k].dtype) for k in s["wrt"]]}


PLAIN = {"conv": _conv, "conv_step": _conv_step, "scan": _scan, "scan_step": _scan_step, "norm": _norm}


# ---- what a pass cannot do without --------------------------------------------------------------
def work(case):
    op, e = case["op"], SIZE[case["dtype"]]
    if op in ("conv", "conv_step"):
        C, W = case["C"], case["W"]
        cells = case["B"] * case.get("T", 1) * C
        n = (case["nseq"] or case["B"]) if op == "conv" else case["B"]
        weights = C * (W + 1) * e
        states = n * (W - 1) * C * e
        if op == "conv_step":
            return dict(bytes=2 * cells * e + 2 * states + weights, flops=(2 * W + 5) * cells)
        if not case["grad"]:
            return dict(bytes=2 * cells * e + (2 if case["state"] else 1) * states + weights, flops=(2 * W + 5) * cells)
        # forward: x in, out written; backward: x and dout in, dx written; weights and states with their gradients
        return dict(bytes=5 * cells * e + 3 * weights + (3 * states if case["state"] else 0),
                    flops=(3 * (2 * W + 5) + 2 * W) * cells)
    if op in ("scan", "scan_step"):
        D, N, G = (case[k] for k in "DNG")
        T = case["B"] * case.get("T", 1)
        cells, cols = T * D, 2 * T * G * N
        n = (case["nseq"] or case["B"]) if op == "scan" else case["B"]
        rows = 3 + bool(case["gate"])
        weights, states = (D * N + 2 * D) * 4, n * D * N * 4
        if op == "scan_step":
            return dict(bytes=(rows * cells + cols) * e + 2 * states + weights, flops=(7 * N + 10) * cells)
        if not case["grad"]:
            return dict(bytes=(rows * cells + cols) * e + (2 if case["state"] else 1) * states + weights,
                        flops=(7 * N + 10) * cells)
        # backward: the forward's inputs and dout in, their gradients written
        return dict(bytes=(rows * cells + cols) * e + (2 * rows * cells - cells + 2 * cols) * e + 3 * weights
                    + (3 * states if case["state"] else 0), flops=(7 * N + 10 + 20 * N + 20) * cells)
    cells = case["N"] * case["S"] * case["C"]
    rows = 2 + (case["act"] == "gate")
    weights = 2 * case["C"] * e if case["affine"] else 0
    if not case["grad"]:
        return dict(bytes=rows * cells * e + weights, flops=12 * cells)
    return dict(bytes=(rows + 2 * rows - 1) * cells * e + 3 * weights, flops=36 * cells)


# ---- the answer in 64 bits ----------------------------------------------------------------------
def exact(case, seed):
    """From the definitions, sequence by sequence and token by token, gradients by differentiating that."""
    s = prepare(case, seed)
    v = {k: x.detach().double() if torch.is_tensor(x) and x.is_floating_point() else x for k, x in s.items()}
    for k in s.get("wrt", ()):
        v[k].requires_grad_(True)
    with torch.set_grad_enabled(bool(case.get("grad"))):
        out, state = EXACT[case["op"]](v, case)
    if case.get("grad"):
        grads = torch.autograd.grad(out, [v[k] for k in s["wrt"]], v["dout"], allow_unused=True)
        return {"out": out.detach(),
                "grad": [torch.zeros_like(v[k]) if g is None else g for k, g in zip(s["wrt"], grads)]}
    return {"out": out} if state is None else {"out": out, "state": state}


def _silu64(x):
    return x / (1 + torch.exp(-x))


def _spans(v, c):
    if v["cu"] is None:
        return [(i, 0, c["T"]) for i in range(c["B"])]
    cu = v["cu"].tolist()
    return [(0, cu[i], cu[i + 1]) for i in range(len(cu) - 1)]


def _conv64(v, c):
    outs, ends = [], []
    for i, (b, t0, t1) in enumerate(_spans(v, c)):
        x = v["x"][b, t0:t1]
        head = v["init"][i] if v["init"] is not None else x.new_zeros(c["W"] - 1, c["C"])
        x = torch.cat([head, x])
        y = sum(x[k:k + t1 - t0] * v["w"][:, k] for k in range(c["W"]))
        y = y + v["b"] if v["b"] is not None else y
        outs.append(_silu64(y) if c["silu"] else y)
        ends.append(x[t1 - t0:].detach())
    return torch.cat(outs).reshape(v["x"].shape), torch.stack(ends)


def _conv_step64(v, c):
    outs = []
    for b in range(c["B"]):
        at = b if v["slots"] is None else int(v["slots"][b])
        x = torch.cat([v["state"][at], v["x"][b:b + 1]])
        y = (x * v["w"].t()).sum(0)
        y = y + v["b"] if v["b"] is not None else y
        outs.append(_silu64(y) if c["silu"] else y)
        v["state"][at] = x[1:]
    return torch.stack(outs), v["state"]


def _token64(h, u, raw, A, Bm, Cm, c):
    """One token of the recurrence: h, A [.., D, N], u and raw (delta with its bias) [.., D], Bm and Cm [.., G, N]."""
    dt = torch.logaddexp(raw, torch.zeros_like(raw))[..., None]
    rep = c["D"] // c["G"]
    h = torch.exp(dt * A) * h + dt * u[..., None] * Bm.repeat_interleave(rep, -2)
    return h, (h * Cm.repeat_interleave(rep, -2)).sum(-1)


def _scan64(v, c):
    raw, ys, ends = v["delta"] + v["bias"], [], []
    if v["cu"] is None:  # all sequences of the batch at once
        h = v["init"] if v["init"] is not None else v["A"].new_zeros(c["B"], c["D"], c["N"])
        for t in range(c["T"]):
            h, y = _token64(h, v["u"][:, t], raw[:, t], v["A"], v["Bm"][:, t], v["Cm"][:, t], c)
            ys.append(y)
        y, end = torch.stack(ys, 1), h
    else:
        for i, (b, t0, t1) in enumerate(_spans(v, c)):
            h = v["init"][i] if v["init"] is not None else v["A"].new_zeros(c["D"], c["N"])
            for t in range(t0, t1):
                h, y = _token64(h, v["u"][b, t], raw[b, t], v["A"], v["Bm"][b, t], v["Cm"][b, t], c)
                ys.append(y)
            ends.append(h)
        y, end = torch.stack(ys).reshape(v["u"].shape), torch.stack(ends)
    y = y + v["D"] * v["u"] if v["D"] is not None else y
    return (y * _silu64(v["z"]) if v["z"] is not None else y), end.detach()


def _scan_step64(v, c):
    at = torch.arange(c["B"], device="cuda") if v["slots"] is None else v["slots"].long()
    h, y = _token64(v["state"][at], v["u"], v["delta"] + v["bias"], v["A"], v["Bm"], v["Cm"], c)
    v["state"][at] = h
    y = y + v["D"] * v["u"] if v["D"] is not None else y
    return (y * _silu64(v["z"]) if v["z"] is not None else y), v["state"]


def _norm64(v, c):
    x = v["x"].reshape(c["N"], c["S"], c["G"], -1).transpose(1, 2)
    var, mean = torch.var_mean(x, (2, 3), unbiased=False, keepdim=True)
    y = ((x - mean) / torch.sqrt(var + 1e-5)).transpose(1, 2).reshape(v["x"].shape)
    y = y * v["w"] + v["b"] if v["w"] is not None else y
    y = _silu64(y) if c["act"] == "silu" else y * _silu64(v["z"]) if c["act"] == "gate" else y
    return y, None


EXACT = {"conv": _conv64, "conv_step": _conv_step64, "scan": _scan64, "scan_step": _scan_step64, "norm": _norm64}
