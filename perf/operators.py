"""Timing cases of the expert-mixture operators: mixing expert weights, grouped dense maps over
ragged rows, and block-scaled fp8 dense maps.

A mixture-of-linear-experts interatomic potential keeps E expert matrices per dense layer and
gives every system of a batch its own weighted mean of them (`mix_experts`); the edges of each
system then go through that system's matrix (`grouped_linear`). `fp8_linear` is the same map with
8-bit operands, a scale for each block of 128, for frozen weights. The widths are those of the
sphere_channels = 128 model: SO(2) convolutions of 6C -> 5C, 8C -> 4C, 4C -> 2C and 4C -> 4C.

`own` False: elementary torch operations in 32 bits (64 for the long sums); `own` True: the
package's operators.
"""
import math

import numpy as np
import torch

own = False

_DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BLOCK = 128


def listed():
    return [
        # one small cluster in a molecular-dynamics loop: a few edges, one system, forward only; latency
        dict(name="grouped-few-edges-bf16", op="grouped", dtype="bf16", T=24, G=1, K=768, N=640, bias="none", train=False),
        # serving a batch of relaxations in the framework's own precision
        dict(name="grouped-batch-fp32", op="grouped", dtype="fp32", T=30000, G=32, K=1024, N=512, bias="shared", train=False),
        # training step of a convolution over the edges of 4,000 atoms in 16 systems
        dict(name="grouped-train-bf16", op="grouped", dtype="bf16", T=120000, G=16, K=768, N=640, bias="shared", train=True),
        # training on many small molecules, some without edges, per-system bias, widths off the tile sizes
        dict(name="grouped-train-molecules-fp16", op="grouped", dtype="fp16", T=50021, G=301, K=520, N=392, bias="group", train=True),
        # fine-tuning in fp32
        dict(name="grouped-train-fp32", op="grouped", dtype="fp32", T=30011, G=8, K=512, N=512, bias="none", train=True),
        # one system's weights at the start of a simulation: the smallest mix, latency
        dict(name="mix-one-system-fp32", op="mix", dtype="fp32", S=1, E=8, N=128, K=128, train=False),
        # the mix of a training batch, with both gradients
        dict(name="mix-train-bf16", op="mix", dtype="bf16", S=64, E=32, N=640, K=768, train=True),
        dict(name="mix-train-many-fp32", op="mix", dtype="fp32", S=128, E=64, N=1024, K=512, train=True),
        # odd numbers of systems and experts, odd matrix size
        dict(name="mix-odd-fp16", op="mix", dtype="fp16", S=37, E=21, N=389, K=263, train=True),
        # a few edges through frozen 8-bit weights: latency
        dict(name="fp8-few-edges-bf16", op="fp8", dtype="bf16", T=8, G=1, K=512, N=512, bias="none", train=False),
        # screening a large system: forward through one frozen matrix
        dict(name="fp8-large-system-bf16", op="fp8", dtype="bf16", T=120000, G=1, K=1024, N=512, bias="shared", train=False),
        # energy and forces of a batch: forward and input gradient through every system's own matrix
        dict(name="fp8-forces-batch-fp32", op="fp8", dtype="fp32", T=40009, G=24, K=768, N=640, bias="shared", train=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    w = _log(rng, lo, hi)
    return w if rng.random() < 0.2 else max(lo, w // 8 * 8)


def draw(rng):
    op = rng.choice(["grouped", "grouped", "mix", "fp8"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "mix":
        while True:
            case = dict(op=op, dtype=dtype, S=_log(rng, 1, 160), E=_log(rng, 2, 96), N=_width(rng, 48, 1024),
                        K=_width(rng, 48, 1024), train=rng.random() < 0.6)
            if case["S"] * case["E"] * case["N"] * case["K"] <= 128 * 64 * 1024 * 512 and \
                    (case["S"] + case["E"]) * case["N"] * case["K"] <= 192 * 1024 * 512:
                return case
    while True:
        case = dict(op=op, dtype=dtype, T=_log(rng, 1, 120000), G=_log(rng, 1, 400), K=_width(rng, 64, 1024),
                    N=_width(rng, 64, 1024), bias=rng.choice(["none", "shared", "group"]), train=rng.random() < 0.6)
        cost = case["T"] * case["N"] * case["K"] * (3 if case["train"] else 1) * (4 if dtype == "fp32" else 1)
        if cost <= 120000 * 768 * 640 * 3 and case["G"] * case["N"] * case["K"] <= 1 << 28:
            return case


# ---- inputs ------------------------------------------------------------------------------------

def _lengths(T, G, seed):
    """Row counts of G systems that sum to T: sizes spread over a factor of about ten, a few systems
    without rows."""
    r = np.random.default_rng(seed)
    w = np.exp(r.normal(0.0, 0.7, G)) * (r.random(G) >= 0.06)
    if w.sum() == 0:
        w[0] = 1.0
    n = np.floor(w / w.sum() * T).astype(np.int64)
    n[int(np.argmax(w))] += T - int(n.sum())
    return [int(v) for v in n]


def _inputs(case, seed):
    dev, dt = torch.device("cuda"), _DT[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)

    def rand(*shape, scale=1.0):
        return torch.randn(*shape, device=dev, generator=g) * scale

    if case["op"] == "mix":
        S, E, N, K = case["S"], case["E"], case["N"], case["K"]
        d = dict(coeff=torch.softmax(rand(S, E, scale=1.5), 1), experts=rand(E, N, K, scale=K ** -0.5).to(dt))
        if case["train"]:
            d["grad"] = rand(S, N, K, scale=1e-2).to(dt)
        return d
    T, G, K, N = case["T"], case["G"], case["K"], case["N"]
    n = _lengths(T, G, seed)
    x = rand(T, K)
    d = dict(x=(x * torch.sigmoid(x)).to(dt), lengths=n,
             offsets=torch.tensor([0] + list(np.cumsum(n)), dtype=torch.int64, device=dev))
    w = rand(G, N, K, scale=K ** -0.5)
    d["w"] = w if case["op"] == "fp8" else w.to(dt)
    if case["bias"] != "none":
        b = rand(N) if case["bias"] == "shared" else rand(G, N)
        d["b"] = b * 0.1 if case["op"] == "fp8" else (b * 0.1).to(dt)
    if case["train"]:
        d["gy"] = rand(T, N, scale=1e-2).to(dt)
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    d["case"] = case
    if case["op"] == "mix":
        if own and case["train"]:
            d["coeff"].requires_grad_(True)
            d["experts"].requires_grad_(True)
        return d
    if case["op"] == "fp8":
        # the frozen weights, laid out once
        if own:
            from flash_uma_b200.fp8 import Fp8Weight
            d["w8"] = Fp8Weight(d["w"])
            if case["train"]:
                d["x"].requires_grad_(True)
        else:
            d["wq"] = _quantised_weight(d["w"])
        return d
    if own and case["train"]:
        for k in ("x", "w", "b"):
            if k in d:
                d[k].requires_grad_(True)
    return d


# ---- one pass -------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"mix": _own_mix, "grouped": _own_grouped, "fp8": _own_fp8}[op](state)
    return {"mix": _plain_mix, "grouped": _plain_grouped, "fp8": _plain_fp8}[op](state)


def _own_mix(s):
    from flash_uma_b200.grouped import mix_experts
    w = mix_experts(s["coeff"], s["experts"])
    if not s["case"]["train"]:
        return [w]
    gc, ge = torch.autograd.grad(w, [s["coeff"], s["experts"]], s["grad"])
    return [w.detach(), gc, ge]


def _own_grouped(s):
    from flash_uma_b200.grouped import grouped_linear
    y = grouped_linear(s["x"], s["w"], s["offsets"], s.get("b"))
    if not s["case"]["train"]:
        return [y]
    wrt = [s["x"], s["w"]] + ([s["b"]] if "b" in s else [])
    return [y.detach(), *torch.autograd.grad(y, wrt, s["gy"])]


def _own_fp8(s):
    from flash_uma_b200.fp8 import fp8_linear
    y = fp8_linear(s["x"], s["w8"], s["offsets"], s.get("b"))
    if not s["case"]["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, [s["x"]], s["gy"])]


def _plain_mix(s):
    c, e = s["coeff"], s["experts"]
    S, E = c.shape
    e2 = e.reshape(E, -1).float()
    w = (c @ e2).to(e.dtype).reshape(S, *e.shape[1:])
    if not s["case"]["train"]:
        return [w]
    g = s["grad"].reshape(S, -1).float()
    # a sum over every element of a matrix: blocks in 32 bits, joined in 64
    gc = torch.zeros(S, E, dtype=torch.float64, device=c.device)
    for a in range(0, e2.shape[1], 8192):
        gc += (g[:, a:a + 8192] @ e2[:, a:a + 8192].t()).double()
    return [w, gc.float(), (c.t() @ g).to(e.dtype).reshape(e.shape)]


def _spans(lengths):
    o = 0
    for g, n in enumerate(lengths):
        if n:
            yield g, o, o + n
        o += n


def _plain_grouped(s):
    x, w, b, train = s["x"], s["w"], s.get("b"), s["case"]["train"]
    dt, G, N = x.dtype, w.shape[0], w.shape[1]
    y = torch.zeros(x.shape[0], N, dtype=dt, device=x.device)
    if train:
        gx, gw = torch.zeros_like(x), torch.zeros_like(w)
        gb = torch.zeros(G, N, dtype=torch.float64, device=x.device)
    for g, a, z in _spans(s["lengths"]):
        xs, ws = x[a:z].float(), w[g].float()
        r = xs @ ws.t()
        if b is not None:
            r = r + (b if b.dim() == 1 else b[g]).float()
        y[a:z] = r.to(dt)
        if train:
            gs = s["gy"][a:z].float()
            gx[a:z] = (gs @ ws).to(dt)
            gw[g] = (gs.t() @ xs).to(dt)
            if b is not None:
                gb[g] = gs.sum(0, dtype=torch.float64)
    if not train:
        return [y]
    out = [y, gx, gw]
    if b is not None:
        out.append((gb.sum(0) if b.dim() == 1 else gb).to(dt))
    return out


def _round_blocks(v, amax):
    """Values of `v` after rounding to e4m3 under the block maxima `amax`: the scale is the smallest
    power of two (at least 2^-126) that brings the block's maximum to 448 or below."""
    m, e = torch.frexp(amax)                       # amax = m 2^e, m in [0.5, 1); 448 = 0.875 2^9
    k = torch.clamp(e - 9 + (m > 0.875).to(e.dtype), min=-126)
    k = torch.where(amax > 0, k, torch.full_like(k, -126))
    return torch.ldexp(torch.ldexp(v, -k).to(torch.float8_e4m3fn).float(), k)


def _quantised_rows(x):
    T, K = x.shape
    Kp = -(-K // _BLOCK) * _BLOCK
    v = torch.zeros(T, Kp, device=x.device)
    v[:, :K] = x.float()
    v = v.reshape(T, -1, _BLOCK)
    return _round_blocks(v, v.abs().amax(2, keepdim=True)).reshape(T, Kp)[:, :K]


def _quantised_weight(w):
    G, N, K = w.shape
    Np, Kp = -(-N // _BLOCK) * _BLOCK, -(-K // _BLOCK) * _BLOCK
    v = torch.zeros(G, Np, Kp, device=w.device)
    v[:, :N, :K] = w
    v = v.reshape(G, Np // _BLOCK, _BLOCK, Kp // _BLOCK, _BLOCK)
    return _round_blocks(v, v.abs().amax((2, 4), keepdim=True)).reshape(G, Np, Kp)[:, :N, :K].contiguous()


def _plain_fp8(s):
    x, wq, b, train = s["x"], s["wq"], s.get("b"), s["case"]["train"]
    y = torch.zeros(x.shape[0], wq.shape[1], dtype=x.dtype, device=x.device)
    xq = _quantised_rows(x)
    if train:
        gx, gq = torch.zeros_like(x), _quantised_rows(s["gy"])
    for g, a, z in _spans(s["lengths"]):
        r = xq[a:z] @ wq[g].t()
        if b is not None:
            r = r + (b if b.dim() == 1 else b[g])
        y[a:z] = r.to(x.dtype)
        if train:
            gx[a:z] = (gq[a:z] @ wq[g]).to(x.dtype)
    return [y, gx] if train else [y]


# ---- work and exact values ---------------------------------------------------------------------------

def work(case):
    b = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "mix":
        S, E, P = case["S"], case["E"], case["N"] * case["K"]
        byts, flops = (S + E) * P * b + S * E * 4, 2 * S * E * P
        if case["train"]:
            byts, flops = byts + (S + E) * P * b + S * E * 4, 3 * flops
        return {"bytes": byts, "flops": flops}
    T, G, K, N = case["T"], case["G"], case["K"], case["N"]
    wb = 1 if case["op"] == "fp8" else b
    bias = {"none": 0, "shared": N, "group": G * N}[case["bias"]] * (4 if case["op"] == "fp8" else b)
    G = min(G, T)                                  # a system without rows needs no weight
    byts, flops = T * (K + N) * b + G * N * K * wb + bias, 2 * T * N * K
    if case["train"]:
        byts += T * (K + N) * b                    # the output's gradient in, the input's gradient out
        flops *= 2
        if case["op"] == "grouped":
            byts += case["G"] * N * K * b + bias   # the weight gradient
            flops += 2 * T * N * K
    return {"bytes": byts, "flops": flops}


def _e4m3(v):
    """Round float64 values, |v| <= 448, to the nearest e4m3 number, ties to even: the step is
    2^(e - 3) for 2^e <= |v| < 2^(e + 1), and 2^-9 below 2^-6."""
    _, e = torch.frexp(v.abs().clamp(min=2.0 ** -6))
    step = torch.ldexp(torch.ones_like(v), e - 4)
    return torch.round(v / step) * step


def _scale64(amax):
    """2^ceil(log2(amax / 448)) by counting: exact at the borders; 2^-126 for tiny or zero maxima."""
    s = torch.full_like(amax, 2.0 ** -126)
    for k in range(-125, 121):
        s = torch.where(amax > 448.0 * 2.0 ** (k - 1), torch.full_like(s, 2.0 ** k), s)
    return s


def _exact_rows(x):
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for a in range(0, x.shape[1], _BLOCK):
        blk = x[:, a:a + _BLOCK].double()
        sc = _scale64(blk.abs().max(dim=1, keepdim=True).values)
        out[:, a:a + _BLOCK] = _e4m3(blk / sc) * sc
    return out


def _exact_weight(w):
    out = torch.empty(w.shape, dtype=torch.float64, device=w.device)
    for n in range(0, w.shape[1], _BLOCK):
        for k in range(0, w.shape[2], _BLOCK):
            blk = w[:, n:n + _BLOCK, k:k + _BLOCK].double()
            sc = _scale64(blk.abs().flatten(1).max(dim=1).values)[:, None, None]
            out[:, n:n + _BLOCK, k:k + _BLOCK] = _e4m3(blk / sc) * sc
    return out


def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "mix":
        c, e = d["coeff"].double(), d["experts"].double()
        out = [torch.einsum("se,enk->snk", c, e)]
        if case["train"]:
            g = d["grad"].double()
            out += [torch.einsum("snk,enk->se", g, e), torch.einsum("se,snk->enk", c, g)]
        return out
    fp8 = case["op"] == "fp8"
    x = _exact_rows(d["x"]) if fp8 else d["x"].double()
    w = _exact_weight(d["w"]) if fp8 else d["w"].double()
    b = d["b"].double() if "b" in d else None
    gy = None
    if case["train"]:
        gy = _exact_rows(d["gy"]) if fp8 else d["gy"].double()
    T, G, N = x.shape[0], w.shape[0], w.shape[1]
    bounds = np.concatenate([[0], np.cumsum(d["lengths"])])
    y = torch.zeros(T, N, dtype=torch.float64, device=x.device)
    gx, gw = torch.zeros_like(x), torch.zeros_like(w)
    gb = torch.zeros(G, N, dtype=torch.float64, device=x.device)
    for g in range(G):
        rows = slice(int(bounds[g]), int(bounds[g + 1]))
        y[rows] = torch.einsum("tk,nk->tn", x[rows], w[g])
        if b is not None:
            y[rows] += b if b.dim() == 1 else b[g]
        if gy is not None:
            gx[rows] = torch.einsum("tn,nk->tk", gy[rows], w[g])
            if not fp8:
                gw[g] = torch.einsum("tn,tk->nk", gy[rows], x[rows])
                gb[g] = gy[rows].sum(0)
    if gy is None:
        return [y]
    if fp8:
        return [y, gx]
    return [y, gx, gw] + ([] if b is None else [gb.sum(0) if b.dim() == 1 else gb])
