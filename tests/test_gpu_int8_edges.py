"""Expert products over 8-bit weights at the edges of what their entry points take: magnitudes from one end of fp32's
range to the other, gradient rows full of ties.  Every result is compared element by element with the definition in 64 bits; what a code next to a border may change is counted there."""
import pytest
import torch

import moe_distributed_training_amd as moe
from oracle import int8_oracle as oracle

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def close(got, want, slack, dtype, what):
    """got within slack of want before it was rounded to dtype (half a step of the type, or of its subnormal numbers)."""
    fi = torch.finfo(dtype)
    got = got.detach().double().cpu()
    assert got.shape == want.shape and not torch.isnan(got).any(), (what, got.shape, want.shape)
    over = (got - want).abs() - 1.01 * slack - (want.abs() + slack) * fi.eps / 2 * 1.01 - fi.smallest_normal * fi.eps
    assert float(over.max()) <= 0, f"{what}: {float(over.max()):.3g} past its bound at {torch.nonzero(over == over.max())[0].tolist()}"


def mlp_weights(E, d, f, seed):
    g = torch.Generator().manual_seed(seed)
    out = []
    for over in (2, 1, 2):                                  # w1, w2, w3
        w = torch.randn(E, f, d, generator=g) * 0.05
        s = w.abs().amax(over, keepdim=True) / 127
        out += [(w / s).round().to(torch.int8), s.squeeze(over)]
    return out


# ---------------------------------------------------------------------------------------------------------------
# magnitudes
# ---------------------------------------------------------------------------------------------------------------
SMALL = [(-56, 0), (-53, -10), (-51, 0), (-45, 30), (-20, -90), (0, -105), (0, 0)]   # powers of two that rows of x and of the gradient are multiplied by


LARGE = [(20, 0), (40, 0), (63, -100)]


@pytest.mark.parametrize("powers", [SMALL, LARGE])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("d,f,per", [(128, 192, 3), (64, 512, 40)])
def test_mlp_rows_of_any_magnitude(dev, d, f, per, gated, powers):
    """h is a product of two projections: rows of 2^-56 give h of about 2^-115, rows of 2^63 of about 2^126, which fp32 and bf16 hold."""
    T, E, k = per * len(powers), 3, 1
    g = torch.Generator().manual_seed(d + per)
    exps = torch.tensor(powers, dtype=torch.float64).repeat_interleave(per, 0)
    x, dout = ((torch.randn(T, d, generator=g).double() * 2.0 ** exps[:, i:i + 1]).to(BF16) for i in (0, 1))
    sei, ssi, eo, gates = oracle.route(T, E, k, 4)
    gates = (gates * 0.75).to(BF16) if gated else None
    w = mlp_weights(E, d, f, f)
    want = oracle.mlp_bounds(x, w, k, sei, ssi, gates, dout)
    assert float(want["y"].abs().max()) < 2.0 ** 127 and float(want["y"].abs().amax(1).min()) > 2.0 ** -120
    xd, gd = x.to(dev).requires_grad_(True), gates.to(dev).requires_grad_(True) if gated else None
    y = moe.fused_expert_mlp_int8(xd, moe.Int8ExpertWeights(*(t.to(dev) for t in w)), k, ssi.to(dev), eo.to(dev), gd)
    close(y, want["y"], want["y_slack"], BF16, "y")
    dx = torch.autograd.grad(y, xd, dout.to(dev))[0]
    close(dx, want["dx"], want["dx_slack"], BF16, "dx")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("T", [24, 700])
def test_linear_rows_up_to_the_end_of_the_range(dev, dtype, gated, T):
    """Results of up to 2^122: the sum of a row of 2^124 times the row's scale alone would leave fp32's range."""
    K, N, E, k = 512, 192, 3, 2
    g = torch.Generator().manual_seed(T)
    power = torch.tensor([0, 60, 72, 100, 115, 122])[torch.arange(T) % 6].double()
    x = (torch.randn(T, K, generator=g).double().clamp(-3, 3) * 2.0 ** power[:, None]).to(dtype)
    w = torch.randint(-127, 128, (E, N, K), generator=g, dtype=torch.int8).transpose(1, 2)
    ws = (torch.rand(E, N, generator=g) + 0.5) * 2.0 ** -16
    sei, ssi, eo, gw = oracle.route(T, E, k, 3)
    gw = gw.to(dtype) if gated else None
    want = oracle.linear(x, w, ws, k, sei, ssi, gw)
    assert 2.0 ** 114 < float(want["y"].abs().max()) < 2.0 ** 126
    y = moe.parallel_linear_int8(x.to(dev), w.to(dev), ws.to(dev), k, sei.to(dev), ssi.to(dev), None, eo.to(dev), gw.to(dev) if gated else None)
    close(y, want["y"], (want["y_terms"] if gated else want["y"].abs()) * (6 + 2 * k) * 2.0 ** -24, dtype, "y")


# ---------------------------------------------------------------------------------------------------------------
# codes of gradient rows
# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("gated", [False, True])
def test_gradient_rows_full_of_ties(dev, dtype, gated):
    """Half of a row's maximum is 63.5 steps: ties go to the even code, whatever the maximum.  Weights that pick single inputs hand the codes out one by one, and a power of
    two as gate and column scale leaves the quotients as they are."""
    K = N = 256
    T = 254
    tops = torch.arange(129, 256, 2).double()                      # odd: half of it is the other side of a tie in any of the types
    top = tops.repeat(4)[:T]
    dout = torch.empty(T, N, dtype=torch.float64)
    dout[:, 0::4], dout[:, 1::4] = top[:, None] / 2, -top[:, None] / 2
    dout[:, 2::4], dout[:, 3::4] = top[:, None] / 4, torch.arange(0, 64).double()
    dout[:, 7] = top
    dout = dout.to(dtype)
    assert torch.equal(dout[:, 0].double(), top / 2)
    w = torch.eye(K, dtype=torch.int8).unsqueeze(0)
    x = torch.ones(T, K, dtype=dtype, device=dev, requires_grad=True)
    idx = torch.arange(T, device=dev)
    gates = torch.full((T, 1), 0.5, dtype=dtype, device=dev) if gated else None
    y = moe.parallel_linear_int8(x, w.to(dev), torch.full((1, N), 0.25, device=dev), 1, torch.zeros_like(idx), idx, None, None, gates)
    dx = torch.autograd.grad(y, x, dout.to(dev))[0]
    c, s, _ = oracle.codes(dout)
    want = c * s.float().double() * (0.125 if gated else 0.25)
    close(dx, want, 4 * 2.0 ** -24 * want.abs(), dtype, "dx")


@pytest.mark.parametrize("dtype,gates_dtype", [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32), (F32, F32)])
def test_gradient_codes_are_those_of_the_exact_products(dev, dtype, gates_dtype):
    """2^20 products of gradient, gate and column scale: a code that lies 2^-22 of a step or more from a border goes to the nearer side.  (A product is held as an fp32 number and its
    error, together off by 2^-46 of it.)"""
    T, K, N, E, k = 1024, 48, 512, 4, 2
    sei, ssi, eo, gw = oracle.route(T, E, k, 12)
    g = torch.Generator().manual_seed(6)
    w = torch.randint(-127, 128, (E, K, N), generator=g, dtype=torch.int8)
    ws = torch.rand(E, N, generator=g) * 1e-3 + 1e-4
    x, dout, gw = torch.randn(T, K, generator=g).to(dtype), torch.randn(T, N, generator=g).to(dtype), gw.to(gates_dtype)
    want = oracle.linear(x, w, ws, k, sei, ssi, gw, dout, near=127 * 2.0 ** -29)
    xd = x.to(dev).requires_grad_(True)
    y = moe.parallel_linear_int8(xd, w.to(dev), ws.to(dev), k, sei.to(dev), ssi.to(dev), None, eo.to(dev), gw.to(dev))
    dx = torch.autograd.grad(y, xd, dout.to(dev))[0]
    close(dx, want["dx"], want["dx_slack"] + want["dx_terms"] * (6 + k) * 2.0 ** -24, dtype, "dx")


# ---------------------------------------------------------------------------------------------------------------
# what a backward pass keeps, rows without columns, scales anywhere
# ---------------------------------------------------------------------------------------------------------------
def test_gates_alone_keep_no_gate_and_up(dev):
    """The gradient of the gate weights needs the rows of y and nothing else of the MLP."""
    T, d, f, E, k = 1024, 64, 4096, 4, 2
    sei, ssi, eo, gw = oracle.route(T, E, k, 0)
    w = moe.Int8ExpertWeights(*(t.to(dev) for t in mlp_weights(E, d, f, 1)))
    g = torch.Generator().manual_seed(1)
    x, dout, ssi, eo = torch.randn(T, d, generator=g).to(BF16).to(dev), torch.randn(T, d, generator=g).to(BF16).to(dev), ssi.to(dev), eo.to(dev)
    both = x.clone().requires_grad_(True), gw.to(dev).requires_grad_(True)
    want = torch.autograd.grad(moe.fused_expert_mlp_int8(both[0], w, k, ssi, eo, both[1]), both[1], dout)[0]
    alone = gw.to(dev).requires_grad_(True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = moe.fused_expert_mlp_int8(x, w, k, ssi, eo, alone)
    held = torch.cuda.memory_allocated() - before
    rows = T * k * d * 4 + T * d * 2                            # y's fp32 rows and the result
    assert held < rows + (1 << 20), f"{held} bytes are held for the backward pass; gate and up would be {2 * T * k * f * 25 // 8}"
    assert torch.equal(torch.autograd.grad(y, alone, dout)[0], want)


@pytest.mark.parametrize("rows", [0, 1, 5])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_of_no_columns(dev, dtype, rows):
    codes, scales = moe.quantize_rows(torch.empty(rows, 0, dtype=dtype, device=dev))
    assert codes.shape == (rows, 0) and codes.dtype == torch.int8
    assert torch.equal(scales.cpu(), torch.zeros(rows))


@pytest.mark.parametrize("gated", [False, True])
def test_weights_of_no_output_columns(dev, gated):
    """An empty sum for every gate, and zeros for the input."""
    T, K, E, k = 6, 64, 3, 2
    sei, ssi, eo, gw = (t.to(dev) for t in oracle.route(T, E, k, 0))
    x = torch.ones(T, K, dtype=BF16, device=dev, requires_grad=True)
    gates = gw.clone().requires_grad_(True) if gated else None
    y = moe.parallel_linear_int8(x, torch.empty(E, K, 0, dtype=torch.int8, device=dev), torch.empty(E, 0, device=dev), k, sei, ssi, None, eo, gates)
    assert y.shape == (T if gated else T * k, 0) and y.dtype == BF16
    got = torch.autograd.grad(y, (x, gates) if gated else (x,), torch.empty_like(y))
    assert all(torch.equal(g, torch.zeros_like(g)) for g in got)


def test_scales_at_any_address(dev):
    """Scales that are part of a larger tensor begin at any multiple of 4 bytes."""
    T, d, f, E, k = 90, 128, 192, 3, 2
    sei, ssi, eo, gates = (t.to(dev) for t in oracle.route(T, E, k, 0))
    w = moe.Int8ExpertWeights(*(t.to(dev) for t in mlp_weights(E, d, f, 1)))

    def moved(t, by):
        big = torch.zeros(t.numel() + by, dtype=t.dtype, device=dev)
        return big[by:].view(t.shape).copy_(t)
    odd = w._replace(w1_scale=moved(w.w1_scale, 1), w2_scale=moved(w.w2_scale, 2), w3_scale=moved(w.w3_scale, 3))
    x = torch.randn(T, d, generator=torch.Generator().manual_seed(1)).to(BF16).to(dev)

    def step(weights):
        a, b = x.clone().requires_grad_(True), gates.clone().requires_grad_(True)
        y = moe.fused_expert_mlp_int8(a, weights, k, ssi, eo, b)
        return [y.detach(), *torch.autograd.grad(y, (a, b), torch.ones_like(y))]
    assert all(torch.equal(a, b) for a, b in zip(step(odd), step(w)))


# ---------------------------------------------------------------------------------------------------------------
# arguments in other forms
# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("ssi_type,eo_type", [(torch.int32, torch.int64), (torch.int64, torch.int32)])
def test_grouped_rows_in_and_a_weighted_sum_out(dev, dtype, ssi_type, eo_type):
    """A down projection: one grouped row per assignment, and each token's rows weighted and summed; index tensors of different types."""
    T, K, N, E, k = 150, 192, 224, 5, 2
    sei, ssi, eo, gw = oracle.route(T, E, k, 1)
    g = torch.Generator().manual_seed(2)
    w = torch.randint(-127, 128, (E, K, N), generator=g, dtype=torch.int8)
    ws = torch.rand(E, N, generator=g) * 1e-3 + 1e-4
    h, dout, gw = torch.randn(T * k, K, generator=g).to(dtype), torch.randn(T, N, generator=g).to(dtype), gw.to(dtype)
    want = oracle.linear(h, w, ws, 1, sei, ssi, gw, dout, grouped_in=True, near=127 * 2.0 ** -29)
    hd, gd = h.to(dev).requires_grad_(True), gw.to(dev).requires_grad_(True)
    y = moe.parallel_linear_int8(hd, w.to(dev), ws.to(dev), 1, sei.to(dev, ssi_type), ssi.to(dev, ssi_type), None, eo.to(dev, eo_type), gd, grouped_in=True)
    got = torch.autograd.grad(y, (hd, gd), dout.to(dev))
    close(y, want["y"], want["y_terms"] * (6 + 2 * k) * 2.0 ** -24, dtype, "y")
    close(got[0], want["dx_rows"], want["dx_slack"] + want["dx_rows"].abs() * 6 * 2.0 ** -24, dtype, "dx")
    close(got[1], want["d_gates"], want["d_gates_terms"] * (N + 7) * 2.0 ** -24, dtype, "d_gates")


def test_one_matrix_for_all_experts(dev):
    """Codes expanded over the experts (a stride of 0), with a scale for each."""
    T, K, N, E = 70, 128, 160, 6
    sei, ssi, eo, _ = (t.to(dev) for t in oracle.route(T, E, 2, 3))
    g = torch.Generator().manual_seed(0)
    w = torch.randint(-127, 128, (1, N, K), generator=g, dtype=torch.int8).to(dev).transpose(1, 2).expand(E, K, N)
    ws, x = (torch.rand(E, N, generator=g) * 1e-3).to(dev), torch.randn(T, K, generator=g).to(BF16).to(dev)
    a, b = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    ya, yb = (moe.parallel_linear_int8(v, c, ws, 2, sei, ssi, None, eo) for v, c in ((a, w), (b, w.contiguous())))
    assert torch.equal(ya, yb)
    assert torch.equal(torch.autograd.grad(ya.sum(), a)[0], torch.autograd.grad(yb.sum(), b)[0])


@pytest.mark.parametrize("order", [(0, 1, 2), (0, 2, 1), (1, 0, 2), (1, 2, 0), (2, 0, 1), (2, 1, 0)])
def test_weights_of_any_order_of_dimensions_become_the_same_codes(dev, order):
    sizes = (3, 70, 50)
    w = torch.randn(sizes, generator=torch.Generator().manual_seed(1)).to(BF16).to(dev)
    back = [order.index(i) for i in range(3)]
    turned = w.permute(order).contiguous().permute(back)
    assert turned.shape == w.shape
    want, got = moe.quantize_expert_weights(w), moe.quantize_expert_weights(turned)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # every second of a larger tensor's columns and rows
    big = torch.randn(3, 140, 100, generator=torch.Generator().manual_seed(2)).to(dev)
    a, b = moe.quantize_expert_weights(big[:, ::2, 1::2]), moe.quantize_expert_weights(big[:, ::2, 1::2].contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_without_autograd_and_in_inference_mode(dev):
    T, d, f, E, k = 40, 128, 192, 3, 2
    block = moe.ScatterMoEBlock(d, f, E, top_k=k, device=dev).quantize_experts()
    x = torch.randn(T, d, generator=torch.Generator().manual_seed(0)).to(BF16).to(dev)
    want = block(x)[0].detach()
    with torch.no_grad():
        assert torch.equal(block(x)[0], want)
    with torch.inference_mode():
        got = block(x.clone())[0]
        assert torch.equal(got, want) and got.is_inference()
        codes, scales = moe.quantize_rows(x)
        assert torch.equal(codes, moe.quantize_rows(x)[0]) and scales.shape == (T,)


def test_graphs_of_one_memory_pool(dev):
    """Two captured calls whose workspaces may be the same memory, replayed in turn."""
    T, d, f, E, k = 3, 1024, 4096, 4, 2                          # few rows: parts of tiles meet in the workspace
    sei, ssi, eo, gates = (t.to(dev) for t in oracle.route(T, E, k, 0))
    w = moe.Int8ExpertWeights(*(t.to(dev) for t in mlp_weights(E, d, f, 1)))
    x = torch.randn(T, d, generator=torch.Generator().manual_seed(1)).to(BF16).to(dev)
    calls = [lambda: moe.fused_expert_mlp_int8(x, w, k, ssi, eo, gates), lambda: moe.fused_expert_mlp_int8(x, w, k, ssi, eo)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in calls:
            c()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs, pool = [], [], None
    for c in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=pool):
            outs.append(c())
        pool = pool or graphs[0].pool()
    for trial, i in enumerate((0, 1, 1, 0, 0, 1)):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(trial)).to(BF16))
        graphs[i].replay()
        torch.cuda.synchronize()
        got = outs[i].clone()
        assert torch.equal(got, calls[i]()), (trial, i)
