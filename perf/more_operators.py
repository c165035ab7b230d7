"""Experts in 4 bits and what goes with them, as measurable cases: one grouped projection over 4-bit weights
(``parallel_linear_fp4``), the whole layer for a few tokens, router included, over 16-bit or 4-bit weights
(``moe_layer_decode``, ``moe_layer_forward_fp4``), and the SwiGLU of a training step that keeps its inputs in 8 bits for
the backward pass (``swiglu_8bit``).

A 4-bit weight is a code of 1 sign, 2 exponent and 1 mantissa bit (0, 0.5, 1, 1.5, 2, 3, 4, 6) times a power of two that it
shares with the 31 others of its group: 32 consecutive inputs of one output.  ``codes`` (E, N, ceil(K / 32) * 16) hold two
codes a byte, the even input in the lower half, ``scales`` (E, N, ceil(K / 32)) the biased exponents of the powers.

``kind``   linear: one projection; layer: router, experts, weighted sum; swiglu: silu(gate) * up
``mode``   fwd: no gradients; train: outputs and gradients
``T``      rows of the input (swiglu: rows of gate and up), ``k`` experts per row, ``E`` experts; linear: ``K`` inputs, ``N``
           outputs of an expert; layer: ``d`` hidden size, ``f`` expert ffn size; swiglu: ``N`` columns
``dtype``  bf16 / fp16 / fp32 of activations; ``bits`` of a layer's expert weights, 16 (the activations' type) or 4
``gates``  weighted sum of a row's k expert outputs; ``skew`` Zipf-like routing, groups of very different sizes
``joint``  swiglu: gate and up are the halves of one matrix's rows, as a joint projection leaves them
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
WIDE = dict(d=4096, f=14336, E=8, k=2)     # the layer of the default benchmark workload
GROUP = 32                                 # inputs that share a scale
BLOCK = 64                                 # columns of gate or up that share a scale


def _linear(name, mode, T, K, N, E, k, dtype="bf16", gates=True, skew=False):
    return dict(name=name, kind="linear", mode=mode, T=T, K=K, N=N, E=E, k=k, dtype=dtype, gates=gates, skew=skew)


def _layer(name, T, d, f, E, k, bits, dtype="bf16"):
    return dict(name=name, kind="layer", mode="fwd", T=T, d=d, f=f, E=E, k=k, bits=bits, dtype=dtype)


def _swiglu(name, mode, T, N, dtype="bf16", joint=False):
    return dict(name=name, kind="swiglu", mode=mode, T=T, N=N, dtype=dtype, joint=joint)


def listed():
    return [
        # one projection for the next token of one sequence: two experts' codes are streamed for one row each
        _linear("linear_one_token", "fwd", 1, 4096, 14336, 8, 2, gates=False),
        # the tiny configuration in fp32: bringing a quantised model up, checking its numerics; launches are all of its time
        _linear("linear_tiny_fp32", "train", 256, 128, 256, 8, 2, "fp32"),
        # one projection of a short prompt, sizes that fill neither a tile nor the last group of inputs
        _linear("linear_odd_fp16", "fwd", 333, 1000, 1368, 8, 2, "fp16"),
        # one projection within a training step: the gradient passes through frozen 4-bit weights
        _linear("linear_train_gates", "train", 1500, 4096, 4096, 8, 2),
        # one projection of a whole sequence of 4096 tokens, prefill or evaluation
        _linear("linear_prefill", "fwd", 4096, 4096, 14336, 8, 2, gates=False),
        # token by token generation for one sequence, expert weights as they are
        _layer("layer_one_token", 1, **WIDE, bits=16),
        # a small model generating for three sequences: launches are all of its time
        _layer("layer_small_fp16", 3, 256, 512, 8, 2, 16, "fp16"),
        # token by token generation for one sequence, experts in 4 bits
        _layer("layer_one_token_fp4", 1, **WIDE, bits=4),
        # generation for sixteen sequences: nearly every expert, a few rows each
        _layer("layer_batch_fp4", 16, **WIDE, bits=4),
        # many narrow experts, wide top-k, eight sequences
        _layer("layer_many_experts_fp4_fp16", 8, 2048, 1024, 64, 8, 4, "fp16"),
        # the activation of one sequence of 4096 tokens (two experts each) within a training step
        _swiglu("swiglu_train", "train", 8192, 14336),
        # the same for a small model, in halves of a joint projection whose width fills no block
        _swiglu("swiglu_train_odd_fp16", "train", 1000, 1368, "fp16", joint=True),
    ]


def _macs(c):
    if c["kind"] == "swiglu":
        return 16 * c["T"] * c["N"]
    R = c["T"] * c["k"]
    if c["kind"] == "layer":
        return R * 3 * c["d"] * c["f"] + c["T"] * c["d"] * c["E"]
    return R * c["K"] * c["N"] * (2 if c["mode"] == "train" else 1)


def _cost(c):
    w = work(c)
    return max(w["bytes"] / 5e12, w["flops"] / 1e15)


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges: projections of even and odd sizes from one row to a long batch, layers of 1 to 16
    tokens from small ones to the wide one, activations from a row to a long batch; never costlier than the largest listed."""
    most = max(_cost(c) for c in listed())
    while True:
        what = rng.choice(["linear", "odd", "wide", "layer", "layer_wide", "layer_many", "swiglu"])
        dt = rng.choice(["bf16", "bf16", "fp16"])
        mode = rng.choice(["fwd", "train"])
        skew = rng.random() < 0.3
        if what in ("linear", "odd"):
            E = rng.randrange(1, 17)
            k = rng.randrange(1, min(E, 4) + 1)
            step = 64 if what == "linear" else 1
            K, N = (step * max(1, _log_int(rng, 64, 5120) // step) for _ in range(2))
            T = _log_int(rng, 1, 8192)
            dt = rng.choice([dt, dt, "fp32"])
            if dt == "fp32":
                T, K, N = min(T, 1024), min(K, 1024), min(N, 1024)
            c = _linear("", mode, T, K, N, E, k, dt, rng.random() < 0.6, skew)
        elif what == "wide":
            c = _linear("", mode, _log_int(rng, 1, 4096), *rng.choice([(4096, 14336), (14336, 4096)]), 8, 2, dt, rng.random() < 0.5, skew)
        elif what == "layer":
            E = rng.randrange(2, 17)
            c = _layer("", rng.randrange(1, 17), 64 * rng.randrange(2, 33), 64 * rng.randrange(2, 49), E, rng.randrange(1, min(E, 4) + 1),
                       rng.choice([16, 4]), dt)
        elif what == "layer_wide":
            c = _layer("", _log_int(rng, 1, 16), **WIDE, bits=rng.choice([16, 4]), dtype=dt)
        elif what == "layer_many":
            c = _layer("", rng.randrange(1, 17), 64 * rng.randrange(8, 41), 64 * rng.randrange(6, 25), rng.choice([16, 32, 64, 96]),
                       rng.randrange(2, 9), rng.choice([16, 4]), dt)
        else:
            c = _swiglu("", mode, _log_int(rng, 1, 16384), _log_int(rng, 32, 14336), rng.choice([dt, dt, "fp32"]), rng.random() < 0.4)
        if _cost(c) <= most:
            del c["name"]
            return c


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _levels(device):
    return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=device)


def _fp4_weights(E, N, K, gen):
    """Codes and scales of N(0, 0.02) weights.  The power of two of a group is the least that leaves its largest magnitude at 7
    of its units or fewer, and every weight becomes the nearest code, the even one of two."""
    G = -(-K // GROUP)
    codes = torch.empty((E, N, G * GROUP // 2), dtype=torch.uint8, device="cuda")
    scales = torch.empty((E, N, G), dtype=torch.uint8, device="cuda")
    for e in range(E):
        w = torch.zeros((N, G * GROUP), device="cuda")
        w[:, :K] = torch.randn((N, K), generator=gen, device="cuda") * 0.02
        w = w.view(N, G, GROUP)
        mantissa, exponent = torch.frexp(w.abs().amax(-1, keepdim=True))
        power = torch.where(mantissa > 0.875, exponent - 2, exponent - 3)
        t = torch.ldexp(w.abs(), -power)
        t = torch.where(t < 2, (2 * t).round() / 2, torch.where(t < 4, t.round(), 2 * (t / 2).round())).clamp(max=6)
        c = torch.bucketize(t, _levels("cuda")) + 8 * (w < 0)
        c = c.view(N, -1, 2)
        codes[e] = (c[..., 0] + 16 * c[..., 1]).to(torch.uint8)
        scales[e] = (power.squeeze(-1) + 127).to(torch.uint8)
    return codes, scales


def _routing(c, gen):
    T, E, k = c["T"], c["E"], c["k"]
    logits = torch.randn((T, E), generator=gen, device="cuda")
    if c["skew"]:
        logits = logits - 1.2 * torch.log(torch.arange(1, E + 1, device="cuda", dtype=torch.float32))
    top, idx = logits.softmax(-1).topk(k, -1)
    sei, ssi = idx.reshape(-1).sort(stable=True)
    offsets = torch.bincount(sei, minlength=E).cumsum(0)
    return sei, ssi, offsets, top / top.sum(-1, keepdim=True)


def _activations(rows, cols, gen):
    """Activations behind a norm: of one size on average, some rows larger than others."""
    size = (0.4 * torch.randn((rows, 1), generator=gen, device="cuda")).exp()
    return size * torch.randn((rows, cols), generator=gen, device="cuda")


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    s = dict(case=c)
    train = c["mode"] == "train"
    if c["kind"] == "swiglu":
        both = _activations(c["T"], 2 * c["N"], gen).to(dt)
        s["gate"], s["up"] = both[:, :c["N"]], both[:, c["N"]:]
        if not c["joint"]:
            s["gate"], s["up"] = s["gate"].contiguous(), s["up"].contiguous()
        if train:
            s["gate"], s["up"] = (s[n].detach().requires_grad_(True) for n in ("gate", "up"))
            s["dout"] = torch.randn((c["T"], c["N"]), generator=gen, device="cuda").to(dt)
        return s
    s["x"] = _activations(c["T"], c["K"] if c["kind"] == "linear" else c["d"], gen).to(dt)
    if c["kind"] == "layer":
        s["wg"] = (torch.randn((c["E"], c["d"]), generator=gen, device="cuda") * 0.02).to(dt)
        for name in ("w1", "w2", "w3"):
            rows, inner = (c["d"], c["f"]) if name == "w2" else (c["f"], c["d"])
            if c["bits"] == 4:
                s[name], s[name + "_scale"] = _fp4_weights(c["E"], rows, inner, gen)
            else:   # all three are kept as (E, f, d)
                s[name] = torch.empty((c["E"], c["f"], c["d"]), dtype=dt, device="cuda")
                for e in range(c["E"]):
                    s[name][e] = torch.randn((c["f"], c["d"]), generator=gen, device="cuda") * 0.02
        return s
    s["sei"], s["ssi"], s["offsets"], gates = _routing(c, gen)
    s["gates"] = gates.to(dt) if c["gates"] else None   # (as a model hands them to its experts: in the activations' type)
    s["codes"], s["scales"] = _fp4_weights(c["E"], c["N"], c["K"], gen)
    if train:
        s["dout"] = torch.randn((c["T"] if c["gates"] else c["T"] * c["k"], c["N"]), generator=gen, device="cuda").to(dt)
        s["x"].requires_grad_(True)
        if c["gates"]:
            s["gates"].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------
def _dequantised(codes, scales, K):
    """(n, N, K) fp32 weights of (n, N, K/2) codes."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()
    v = _levels(codes.device)[(c & 7).long()]
    v = torch.where(c >= 8, -v, v).view(*scales.shape, GROUP)
    return torch.ldexp(v, scales.int().unsqueeze(-1) - 127).flatten(-2)[..., :K]


def _grouped(sei, offsets, rows, weights, transposed):
    """Rows of the grouped order times their expert's matrix: the groups side by side, padded to the longest, and one batched
    product over the experts that have rows.  weights(used): their matrices in fp32."""
    counts = torch.diff(offsets, prepend=offsets.new_zeros(1))
    used = counts.nonzero().squeeze(1)
    slot = torch.zeros_like(counts).index_put_((used,), torch.arange(used.numel(), device=used.device))[sei]
    place = torch.arange(rows.size(0), device=rows.device) - (offsets - counts)[sei]
    padded = rows.new_zeros((used.numel(), int(counts.max()), rows.size(1)))
    padded[slot, place] = rows
    m = weights(used)
    return torch.bmm(padded, m.transpose(1, 2).contiguous() if transposed else m.contiguous())[slot, place]


def _unsorted(ssi, rows):
    out = torch.empty_like(rows)
    out[ssi] = rows
    return out


def _plain_linear(s):
    c, sei, ssi, offsets, k = s["case"], s["sei"], s["ssi"], s["offsets"], s["case"]["k"]
    dt = s["x"].dtype

    def weights(used):
        return _dequantised(s["codes"][used], s["scales"][used], c["K"])
    y = _unsorted(ssi, _grouped(sei, offsets, s["x"].detach().float()[ssi // k], weights, True))
    gates = s["gates"].detach().float() if c["gates"] else None
    out = [((gates.unsqueeze(-1) * y.view(c["T"], k, -1)).sum(1) if c["gates"] else y).to(dt)]
    if c["mode"] == "train":
        g = s["dout"].float()
        rows = g[ssi // k] * gates.reshape(-1)[ssi][:, None] if c["gates"] else g[ssi]
        out.append(_unsorted(ssi, _grouped(sei, offsets, rows, weights, False)).view(c["T"], k, -1).sum(1).to(dt))
        if c["gates"]:
            out.append((y.view(c["T"], k, -1) * g.unsqueeze(1)).sum(-1).to(dt))
    return out


def _plain_layer(s):
    c, x, k = s["case"], s["x"].float(), s["case"]["k"]
    # (choices between experts are values next to a border: logits in 64 bits, ties to the lower expert)
    scores = torch.matmul(s["x"].double(), s["wg"].double().t()).softmax(-1)
    top, idx = scores.sort(dim=-1, descending=True, stable=True)
    top, idx = top[:, :k].float(), idx[:, :k]
    top = top / top.sum(-1, keepdim=True)
    sei, ssi = idx.reshape(-1).sort(stable=True)
    offsets = torch.bincount(sei, minlength=c["E"]).cumsum(0)

    def weights(name, inner):
        if c["bits"] == 16:
            return lambda used: s[name][used].float()
        return lambda used: _dequantised(s[name][used], s[name + "_scale"][used], inner)
    rows = x[ssi // k]
    gate = _grouped(sei, offsets, rows, weights("w1", c["d"]), True)
    up = _grouped(sei, offsets, rows, weights("w3", c["d"]), True)
    h = gate / (1 + torch.exp(-gate)) * up
    y = _unsorted(ssi, _grouped(sei, offsets, h, weights("w2", c["f"]), c["bits"] == 4))
    return [(top.unsqueeze(-1) * y.view(c["T"], k, -1)).sum(1).to(s["x"].dtype), top, idx.int()]


def _kept(v):
    """v as its 8-bit codes give it back: blocks of 64 columns, 127 steps to a block's largest magnitude.  The quotient that is
    rounded is taken in 64 bits: a code is a value next to a border."""
    rows, cols = v.shape
    v = torch.nn.functional.pad(v.double(), (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    a = v.abs().amax(-1, keepdim=True)
    q = torch.where(a > 0, 127 * v / a, torch.zeros_like(v)).round()
    return (q.float() * (a / 127).float()).view(rows, -1)[:, :cols]


def _plain_swiglu(s):
    gate, up = s["gate"].detach(), s["up"].detach()
    g = gate.float()
    out = [(g / (1 + torch.exp(-g)) * up.float()).to(gate.dtype)]
    if s["case"]["mode"] == "train":
        g, u, dh = _kept(gate), _kept(up), s["dout"].float()
        sig = 1 / (1 + torch.exp(-g))
        out += [(dh * u * sig * (1 + g * (1 - sig))).to(gate.dtype), (dh * g * sig).to(gate.dtype)]
    return out


def run(state):
    s = state
    c = s["case"]
    if not own:
        return {"linear": _plain_linear, "layer": _plain_layer, "swiglu": _plain_swiglu}[c["kind"]](s)
    import moe_distributed_training_amd as moe
    with torch.set_grad_enabled(c["mode"] == "train"):
        if c["kind"] == "layer":
            if c["bits"] == 16:
                return list(moe.moe_layer_decode(s["x"], s["wg"], s["w1"], s["w2"], s["w3"], c["k"]))
            weights = moe.Fp4ExpertWeights(s["w1"], s["w1_scale"], s["w2"], s["w2_scale"], s["w3"], s["w3_scale"])
            return list(moe.moe_layer_forward_fp4(s["x"], s["wg"], weights, c["k"]))
        if c["kind"] == "linear":
            y = moe.parallel_linear_fp4(s["x"], s["codes"], s["scales"], c["k"], s["sei"], s["ssi"], None, s["offsets"], s["gates"])
            wanted = [s["x"]] if s["gates"] is None else [s["x"], s["gates"]]
        else:
            y = moe.swiglu_8bit(s["gate"], s["up"])
            wanted = [s["gate"], s["up"]]
    if c["mode"] == "fwd":
        return [y]
    return [y.detach(), *torch.autograd.grad(y, wanted, s["dout"])]


# ---------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def _exact_matrix(codes, scales, K):
    """One expert's (N, K) matrix in 64 bits, digit by digit."""
    nibbles = torch.empty((codes.size(0), codes.size(1) * 2), dtype=torch.int64, device=codes.device)
    nibbles[:, 0::2] = (codes % 16).long()
    nibbles[:, 1::2] = torch.div(codes, 16, rounding_mode="floor").long()
    e, m = (nibbles // 2) % 4, (nibbles % 2).double()
    magnitude = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.pow(2.0, (e - 1).double()))
    power = torch.pow(2.0, scales.double() - 127).repeat_interleave(GROUP, dim=1)
    return (torch.where(nibbles >= 8, -1.0, 1.0) * magnitude * power)[:, :K]


def _exact_linear(case, s):
    c, k, T = case, case["k"], case["T"]
    x = s["x"].detach().double()
    train = c["mode"] == "train"
    gates = s["gates"].detach().double() if c["gates"] else None
    y = torch.zeros((T * k, c["N"]), dtype=torch.float64, device="cuda")
    dx = torch.zeros((T * k, c["K"]), dtype=torch.float64, device="cuda")
    for e in range(c["E"]):
        p = s["ssi"][s["sei"] == e]                       # flat positions that chose this expert
        if p.numel() == 0:
            continue
        w = _exact_matrix(s["codes"][e], s["scales"][e], c["K"])
        token = torch.div(p, k, rounding_mode="floor")
        y[p] = torch.matmul(x[token], w.t())
        if train:
            dy = s["dout"].double()
            dx[p] = torch.matmul(dy[token] * gates.reshape(-1)[p, None] if c["gates"] else dy[p], w)
    y3 = y.view(T, k, -1)
    out = [torch.einsum("tkn,tk->tn", y3, gates) if c["gates"] else y]
    if train:
        out.append(dx.view(T, k, -1).sum(dim=1))
        if c["gates"]:
            out.append(torch.einsum("tkn,tn->tk", y3, s["dout"].double()))
    return out


def _exact_layer(case, s):
    c = case
    x = s["x"].double()
    logits = torch.matmul(x, s["wg"].double().t())
    p = torch.exp(logits - logits.amax(1, keepdim=True))
    order = torch.argsort(p, dim=1, descending=True, stable=True)[:, :c["k"]]
    w = torch.gather(p, 1, order)
    w = w / w.sum(dim=1, keepdim=True)
    out = torch.zeros_like(x)
    for e in range(c["E"]):
        t, j = torch.nonzero(order == e, as_tuple=True)
        if t.numel() == 0:
            continue
        if c["bits"] == 4:
            w1, w3 = (_exact_matrix(s[n][e], s[n + "_scale"][e], c["d"]) for n in ("w1", "w3"))
            w2 = _exact_matrix(s["w2"][e], s["w2_scale"][e], c["f"]).t()
        else:
            w1, w2, w3 = (s[n][e].double() for n in ("w1", "w2", "w3"))
        a, b = torch.matmul(x[t], w1.t()), torch.matmul(x[t], w3.t())
        out[t] += w[t, j, None] * torch.matmul(a * torch.sigmoid(a) * b, w2)
    return [out, w, order.int()]


def _exact_kept(v):
    out = torch.empty_like(v)
    for at in range(0, v.size(1), BLOCK):
        b = v[:, at:at + BLOCK]
        top = b.abs().max(dim=1, keepdim=True).values
        out[:, at:at + BLOCK] = torch.round(torch.nan_to_num(b * 127 / top, nan=0.0)) * (top / 127)
    return out


def _exact_swiglu(case, s):
    g, u = s["gate"].detach().double(), s["up"].detach().double()
    out = [g * torch.sigmoid(g) * u]
    if case["mode"] == "train":
        g, u, dh = _exact_kept(g), _exact_kept(u), s["dout"].double()
        z = torch.sigmoid(g)
        out += [dh * u * (z + g * z * (1 - z)), dh * g * z]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "layer": _exact_layer, "swiglu": _exact_swiglu}[case["kind"]](case, s)


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def _experts_touched(c):
    T, E, k = c["T"], c["E"], c["k"]
    return min(T * k, E * (1.0 - (1.0 - k / E) ** T)) if E > 1 else 1.0


def work(case):
    """Inputs, weights of the experts that rows reach, indices and gate weights read once; outputs and gradients written once.
    (The backward pass of a projection reads the weights again, that of the activation the 8-bit copies that the forward pass
    wrote: neither is counted.)"""
    c = case
    b = torch.finfo(DTYPES[c["dtype"]]).bits // 8
    if c["kind"] == "swiglu":
        return {"bytes": float(c["T"] * c["N"] * b * (3 if c["mode"] == "fwd" else 6)), "flops": float(c["T"] * c["N"] * (6 if c["mode"] == "fwd" else 24))}
    R, used = c["T"] * c["k"], _experts_touched(c)
    if c["kind"] == "layer":
        each = 2 * 3 * c["d"] * c["f"] if c["bits"] == 16 else 3 * c["d"] * c["f"] * 17 / 32
        return {"bytes": float(used * each + c["E"] * c["d"] * b + 2 * c["T"] * c["d"] * b + 8 * R), "flops": 2.0 * _macs(c)}
    out_rows = c["T"] if c["gates"] else R
    n = c["T"] * c["K"] * b + used * c["N"] * -(-c["K"] // GROUP) * 17 + out_rows * c["N"] * b + 8 * (R + c["E"]) + (b * R if c["gates"] else 0)
    if c["mode"] == "train":
        n += out_rows * c["N"] * b + c["T"] * c["K"] * b + (b * R if c["gates"] else 0)
    return {"bytes": float(n), "flops": 2.0 * _macs(c)}
