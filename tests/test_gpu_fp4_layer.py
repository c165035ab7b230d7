"""Expert MLP, layer and block over 4-bit weights: against the composition of their parts (which are tested against 64 bits on their own), against 64 bits, and
used together: an expert layer is trained around frozen 4-bit experts, then serves single tokens.

The MLP in fp32 against 64 bits: with the constants below, every error is first order, at most (terms + 16) 2^-24 of the magnitudes of a sum's terms, carried through the
formulas' derivatives: |silu| <= |g|, |silu'| <= 1.1, |silu''| <= 0.5."""
import pytest
import torch

import moe_distributed_training_amd as moe
from moe_distributed_training_amd._lib import entry
from oracle import fp4_oracle as oracle

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def make(dev, T, d, f, E, k, dtype, seed=0, spread=0.05):
    g = torch.Generator().manual_seed(seed * 7 + T + d + f)
    x = torch.randn(T, d, generator=g).to(dtype)
    wg = (torch.randn(E, d, generator=g) * 0.1).to(dtype)
    w = [torch.randn(E, f, d, generator=g) * spread for _ in range(3)]
    q = moe.Fp4ExpertWeights.quantize(*(t.to(dev) for t in w))
    sei, ssi, offs, gates = oracle.route(T, E, k, seed)
    return x.to(dev), wg.to(dev), q, (sei.to(dev), ssi.to(dev), offs.to(dev), gates.to(dev, dtype))


def exact(q, d, f):
    return [oracle.weights(c.cpu(), s.cpu(), n) for c, s, n in ((q.w1, q.w1_scale, d), (q.w2, q.w2_scale, f), (q.w3, q.w3_scale, d))]


def test_weights_from_storage(dev):
    g = torch.Generator().manual_seed(0)
    w = [torch.randn(3, 72, 40, generator=g).to(BF16) for _ in range(3)]
    a = moe.Fp4ExpertWeights.quantize(*(t.to(dev) for t in w))
    b = moe.Fp4ExpertWeights.quantize(*(t.view(3 * 72, 40).to(dev) for t in w), 72, 40)
    want = [t for v in (oracle.quantize(w[0].transpose(1, 2)), oracle.quantize(w[1]), oracle.quantize(w[2].transpose(1, 2))) for t in v]
    for u, v, n in zip(a, b, want):
        assert torch.equal(u, v) and torch.equal(u.cpu(), n)


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,d,f,E,k", [(1, 64, 64, 2, 2), (9, 100, 72, 3, 2), (70, 256, 384, 4, 1), (300, 128, 200, 5, 3)])
def test_mlp_is_its_parts(dev, T, d, f, E, k, dtype, keep):
    x, _, q, (sei, ssi, offs, gates) = make(dev, T, d, f, E, k, dtype)
    a, b = x.requires_grad_(True), gates.requires_grad_(True)
    lin = lambda v, c, s, kk, g, gi, go: moe.parallel_linear_fp4(v, c, s, kk, sei, ssi, None, offs, g, gi, go)

    def parts(gates, grouped_out):
        g, u = lin(a, q.w1, q.w1_scale, k, None, False, True), lin(a, q.w3, q.w3_scale, k, None, False, True)
        return lin(moe.swiglu_8bit(g, u) if keep else entry("swiglu")(g, u), q.w2, q.w2_scale, 1, gates, True, grouped_out)
    for gw, go in ((b, False), (None, False), (None, True)):
        y, want = moe.fused_expert_mlp_fp4(a, q, k, ssi, offs, gw, go, keep), parts(gw, go)
        assert torch.equal(y, want)
        with torch.no_grad():
            assert torch.equal(moe.fused_expert_mlp_fp4(a, q, k, ssi, offs, gw, go, keep), want)
        leaves = [a] + ([b] if gw is not None else [])
        dout = torch.randn(y.shape, generator=torch.Generator().manual_seed(3)).to(dev, dtype)
        assert all(torch.equal(u, v) for u, v in zip(torch.autograd.grad(y, leaves, dout), torch.autograd.grad(want, leaves, dout)))


def test_mlp_in_fp32_against_64_bits(dev):
    T, d, f, E, k = 40, 96, 136, 4, 2
    x, _, q, (sei, ssi, offs, gates) = make(dev, T, d, f, E, k, F32)
    w1, w2, w3 = exact(q, d, f)
    a, b = x.requires_grad_(True), gates.requires_grad_(True)
    y = moe.fused_expert_mlp_fp4(a, q, k, ssi, offs, b)
    dout = torch.randn(T, d, generator=torch.Generator().manual_seed(3))
    dx, dg = torch.autograd.grad(y, (a, b), dout.to(dev))
    expert = torch.empty(T * k, dtype=torch.long)
    expert[ssi.cpu()] = sei.cpu().long()
    expert = expert.view(T, k)
    xv, gv, D, u = x.detach().double().cpu(), gates.detach().double().cpu(), dout.double(), 2.0 ** -24
    ex, eg = xv.clone().requires_grad_(True), gv.clone().requires_grad_(True)
    rows = torch.stack([torch.stack([w2[e] @ (torch.nn.functional.silu(w1[e] @ ex[t]) * (w3[e] @ ex[t])) for e in expert[t].tolist()]) for t in range(T)])
    ey = (rows * eg.unsqueeze(-1)).sum(1)
    edx, edg = torch.autograd.grad(ey, (ex, eg), D)
    ys, dxs, dgs = torch.zeros(T, d).double(), torch.zeros(T, d).double(), torch.zeros(T, k).double()
    for t in range(T):
        for j, e in enumerate(expert[t].tolist()):
            gt, ut = w1[e].abs() @ xv[t].abs(), w3[e].abs() @ xv[t].abs()
            eh = (d + 16) * 3.2 * gt * ut                                                         # of h, in units of 2^-24
            er = w2[e].abs() @ eh + (f + 16) * (w2[e].abs() @ (gt * ut))                          # of an expert's row
            ys[t] += gv[t, j].abs() * er + (k + 2) * gv[t, j].abs() * rows[t, j].abs().detach()
            dgs[t, j] = D[t].abs() @ er + (d + 16) * (D[t].abs() @ rows[t, j].abs().detach())
            dh = gv[t, j].abs() * (w2[e].abs().t() @ D[t].abs())
            edgate, edup = (d + 24) * dh * ut * (1.1 + 1.1 + 0.5 * gt), (d + 24) * dh * gt * 2.1
            dxs[t] += w1[e].abs().t() @ (edgate + (f + 16) * 1.1 * dh * ut) + w3[e].abs().t() @ (edup + (f + 16) * dh * gt)
    for got, want, bound, what in ((y, ey, ys, "y"), (dx, edx, dxs, "dx"), (dg, edg, dgs, "d_gates")):
        over = (got.detach().double().cpu() - want.detach()).abs() - u * (bound + 4 * want.detach().abs())
        assert float(over.max()) <= 0, what


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("T,dtype", [(5, BF16), (60, F16), (33, F32)])
def test_layer_trains_as_router_and_mlp(dev, T, dtype, normalize, keep):
    d, f, E, k = 128, 192, 4, 2
    x, wg, q, _ = make(dev, T, d, f, E, k, dtype)
    a, b = x.requires_grad_(True), wg.requires_grad_(True)
    out, ew, ei = moe.moe_layer_forward_fp4(a, b, q, k, normalize, keep)
    _, weights, indices = entry("router")(a, b, k, normalize)
    sei, ssi = moe.flatten_and_sort(indices.reshape(-1).long())
    offs = torch.bincount(sei, minlength=E).cumsum(0)
    want = moe.fused_expert_mlp_fp4(a, q, k, ssi, offs, weights, False, keep)
    assert torch.equal(ei.long(), indices.long()) and torch.equal(ew, weights) and torch.equal(out, want)
    dout = torch.randn(out.shape, generator=torch.Generator().manual_seed(3)).to(dev, dtype)
    for u, v in zip(torch.autograd.grad(out, (a, b), dout), torch.autograd.grad(want, (a, b), dout)):
        assert torch.equal(u, v)


def test_layer_gradient_against_differences(dev):
    """fp32, a direction of x and one of the router weight: the slope of a fixed weighting of the outputs over a step h.  The formula's own error over the step is third
    order; outputs are off by about 2^-20 of their size each way (sums of some hundred terms), which over a step of 2^-6 is 2^-13 of slopes of the outputs' size."""
    T, d, f, E, k = 20, 64, 96, 4, 2
    x, wg, q, _ = make(dev, T, d, f, E, k, F32, spread=0.15)
    g = torch.Generator().manual_seed(5)
    dout = torch.randn(T, d, generator=g).to(dev)
    a, b = x.requires_grad_(True), wg.requires_grad_(True)
    out, _, ei = moe.moe_layer_forward_fp4(a, b, q, k)
    grads = torch.autograd.grad(out, (a, b), dout)
    for i in range(2):
        v = torch.randn((x, wg)[i].shape, generator=g).to(dev) * (0.1 if i == 0 else 0.01)
        h = 2.0 ** -6

        def at(s):
            with torch.no_grad():
                o, _, idx = moe.moe_layer_forward_fp4(a + s * v if i == 0 else a, b + s * v if i == 1 else b, q, k)
            assert torch.equal(idx, ei)                                    # (the slope is that of one choice of experts)
            return (o.double() * dout.double()).sum()
        slope = (8 * (at(h) - at(-h)) - (at(2 * h) - at(-2 * h))) / (12 * h)
        want = (grads[i].double() * v.double()).sum()
        size = float(out.detach().double().norm() * dout.double().norm() / (T * d) ** 0.5)
        assert abs(float(slope - want)) <= 2.0 ** -13 * (abs(float(want)) + size)


def test_what_the_backward_pass_keeps(dev):
    """Memory between the passes: gate and up in 2.125 bytes per value of a pair's two against 4."""
    T, d, f, E, k = 2048, 256, 1024, 4, 2
    x, _, q, (sei, ssi, offs, gates) = make(dev, T, d, f, E, k, BF16)
    a = x.requires_grad_(True)
    held = []
    for keep in (False, True):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = moe.fused_expert_mlp_fp4(a, q, k, ssi, offs, gates, False, keep)
        held.append(torch.cuda.memory_allocated() - before - y.numel() * 2)
        del y
    assert held[0] >= T * k * f * 4 and held[1] <= T * k * f * 2.125 + 65536


@pytest.mark.parametrize("lora", [False, True])
@pytest.mark.parametrize("ep", [True, False])
def test_caller_with_8_bit_interims(dev, ep, lora):
    """scattermoe_permute_and_compute(keep_8bit=True) is its three projections around swiglu_8bit."""
    T, d, f, E, k, r = 50, 128, 192, 4, 2, 8
    g = torch.Generator().manual_seed(0)
    w = [(torch.randn(E * f, d, generator=g) * 0.05).to(BF16).to(dev).requires_grad_(not lora) for _ in range(3)]
    sei, ssi, offs, _ = (t.to(dev) for t in oracle.route(T, E, k, 0))
    x = torch.randn(T * k if ep else T, d, generator=g).to(BF16).to(dev).requires_grad_(True)
    views = None
    if lora:
        fac = [(torch.randn(E, *s, generator=g) * 0.1).to(BF16).to(dev).requires_grad_(True) for s in ((d, r), (r, f), (d, r), (r, f), (f, r), (r, d))]
        views = moe.megablocks_utils.moe_mlp.LoraViews(*fac)
    call = lambda keep: moe.scattermoe_permute_and_compute(x, *w, f, d, k, sei, ssi, E, None, ep, offs, views, 16.0, keep)
    fan = 1 if ep else k
    W = [t.view(E, f, d) for t in w]

    def proj(v, i, kk, gi, go):
        view = W[1] if i == 1 else W[i].transpose(1, 2)
        if not lora:
            return moe.parallel_linear(v, view, kk, sei, ssi, None, offs, None, gi, go)
        n = (0, 4, 2)[i]
        return moe.parallel_linear_lora(v, view, fac[n], fac[n + 1], r, 16.0, kk, sei, ssi, None, offs, None, gi, go)
    want = proj(moe.swiglu_8bit(proj(x, 0, fan, False, True), proj(x, 2, fan, False, True)), 1, 1, True, not ep)
    got = call(True)
    assert torch.equal(got, want)
    leaves = [x] + (fac if lora else w)
    dout = torch.randn(got.shape, generator=g).to(BF16).to(dev)
    assert all(torch.equal(u, v) for u, v in zip(torch.autograd.grad(got, leaves, dout), torch.autograd.grad(want, leaves, dout)))
    # near the caller without it: roundings of the interims, and gradients within the codes' 1/254
    plain = call(False)
    assert float((got - plain).detach().float().norm() / plain.detach().float().norm()) <= 4 * 2.0 ** -8
    gp, gk = torch.autograd.grad(plain, x, dout)[0].float(), torch.autograd.grad(call(True), x, dout)[0].float()
    assert float((gp - gk).norm() / gp.norm()) <= 0.03     # block maxima are up to 4 deviations: steps of 4 / 127, uniform errors of 4 / 127 / 12^0.5 = 0.9 % in each of two factors, and roundings


# ---------------------------------------------------------------------------------------------------------------
# blocks
# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_block_in_4_bits(dev, dtype):
    torch.manual_seed(0)
    block = moe.ScatterMoEBlock(128, 192, 4, dtype=dtype, device=dev, bias=True)
    q = moe.Fp4ExpertWeights.quantize(block.w1, block.w2, block.w3, 192, 128)
    assert block.quantize_experts(bits=4) is block and block.expert_bits == 4 and [n for n, _ in block.named_parameters()] == ["bias", "router"]
    for n, t in q._asdict().items():
        assert torch.equal(getattr(block, n), t)
    for shape in ((3, 128), (2, 30, 128), (1, 1, 128)):
        x = torch.randn(shape, generator=torch.Generator().manual_seed(1)).to(dev, dtype)
        with torch.no_grad():
            want = moe.moe_layer_forward_fp4(x.reshape(-1, 128), block.router, q)[0].view(shape)
            assert torch.equal(block(x), want) and torch.equal(block.decode(x), want)
    # the gradients of the router and of the input; 8-bit interims from now on
    x.requires_grad_(True)
    block.quantize_experts(bits=4, keep_8bit=True)
    block(x).sum().backward()
    want = torch.autograd.grad(moe.moe_layer_forward_fp4(x.reshape(-1, 128), block.router, q, keep_8bit=True)[0].view(shape).sum(), (x, block.router))
    assert torch.equal(x.grad, want[0]) and torch.equal(block.router.grad, want[1])


def test_block_in_4_bits_is_saved_and_loaded(dev):
    torch.manual_seed(0)
    a = moe.ScatterMoEBlock(64, 128, 3, device=dev).quantize_experts(bits=4)
    torch.manual_seed(1)
    b = moe.ScatterMoEBlock(64, 128, 3, device=dev).quantize_experts(bits=4)
    x = torch.randn(20, 64, generator=torch.Generator().manual_seed(1)).to(BF16).to(dev)
    with torch.no_grad():
        assert not torch.equal(a(x)[0], b(x)[0])
        b.load_state_dict(a.state_dict())
        assert torch.equal(a(x)[0], b(x)[0])
        c = b.float()
        assert c(x.float())[0].dtype == F32                                  # codes serve any of the three types


def test_decode_of_a_block(dev):
    torch.manual_seed(0)
    block = moe.ScatterMoEBlock(128, 192, 4, device=dev)
    x = torch.randn(2, 3, 128, generator=torch.Generator().manual_seed(1)).to(BF16).to(dev)
    out, none = block.decode(x)
    assert none is None and out.shape == x.shape and not out.requires_grad
    w = [t.detach().view(4, 192, 128) for t in (block.w1, block.w2, block.w3)]
    with torch.no_grad():
        assert torch.equal(out.view(6, 128), moe.moe_layer_decode(x.view(6, 128), block.router, *w)[0])
    with pytest.raises(RuntimeError, match="up to 16 tokens"):
        block.decode(torch.zeros(17, 128, dtype=BF16, device=dev))


def test_trained_around_4_bit_experts_then_serving_tokens(dev):
    """The operators as they are used: experts into 4 bits; steps of router and input projection through the layer with 8-bit interims, captured into a graph; then tokens one by
    one and in small batches, which agree with the layer for many tokens."""
    d, f, E, k, T = 128, 256, 6, 2, 96
    torch.manual_seed(0)
    block = moe.ScatterMoEBlock(d, f, E, top_k=k, device=dev).quantize_experts(bits=4, keep_8bit=True)
    front = torch.nn.Linear(d, d, device=dev, dtype=BF16)
    params = [*front.parameters(), block.router]
    x, target = (torch.randn(T, d, generator=torch.Generator().manual_seed(i)).to(BF16).to(dev) for i in range(2))

    def step():
        for p in params:
            p.grad = None
        ((block(front(x))[0] - target).float() ** 2).sum().backward()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    captured = [p.grad for p in params]
    for n in range(4):
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        step()
        assert all(bool(torch.isfinite(u).all()) and torch.equal(u, p.grad) for u, p in zip(got, params)), n
        with torch.no_grad():
            for p, u in zip(params, got):
                p -= 1e-4 * u
    with torch.no_grad():
        h = front(x)
        many = block(h)[0]
        for rows in ([0], [5], list(range(16)), [95, 3, 3]):
            few = block.decode(h[rows])[0]
            # the layer for many tokens rounds gate, up and h to the type, a half step each, this one does not
            assert float((few.float() - many[rows].float()).norm() / many[rows].float().norm()) <= 4 * 2.0 ** -8


def test_decode_of_blocks_in_8_bits_and_with_a_bias(dev):
    x = torch.randn(5, 128, generator=torch.Generator().manual_seed(1)).to(BF16).to(dev)
    for bits in (8, 4, 16):
        torch.manual_seed(0)
        block = moe.ScatterMoEBlock(128, 192, 4, device=dev, bias=True, return_bias=True)
        if bits != 16:
            block.quantize_experts(bits=bits)
        with torch.no_grad():
            out, bias = block.decode(x)
            want, _ = block(x)
        assert bias is block.bias and out.shape == x.shape
        if bits != 16:
            assert torch.equal(out, want)
        assert float((out.float() - want.float()).norm() / want.float().norm()) <= 4 * 2.0 ** -8
        assert block.decode(x[:0])[0].shape == (0, 128)
