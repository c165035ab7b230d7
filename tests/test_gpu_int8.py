"""Expert products over 8-bit weights against their definition in 64 bits.

Sums of codes are exact, so a projection's result is off by its last rounding (half a step of its type) and the fp32 roundings of
the two scales, of the sum and of their products (six of 2^-24), element by element.  Where codes are taken of computed values
(gradients, h), a value next to a border may round the other way: the oracle says what those can change."""
import pytest
import torch

import moe_distributed_training_amd as moe
from oracle import int8_oracle as oracle

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
F32_STEPS = 6 * 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, slack, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    over = (got - want).abs() - slack
    assert not torch.isnan(got).any(), f"{what}: NaN"
    assert float(over.max()) <= 0, f"{what}: {float(over.max()):.3g} past its bound at {torch.nonzero(over == over.max())[0].tolist()}"


def norm_rel(got, want):
    return float((got.detach().double().cpu() - want).norm() / want.norm())


# ---------------------------------------------------------------------------------------------------------------
# rows and weights into codes
# ---------------------------------------------------------------------------------------------------------------
def check_rows(x, dev):
    c, s, _ = oracle.codes(x)
    q, scale = moe.quantize_rows(x.to(dev))
    assert q.dtype == torch.int8 and scale.dtype == F32 and q.shape == x.shape
    assert torch.equal(q.cpu().double(), c), "codes differ"
    assert torch.equal(torch.nan_to_num(scale.cpu(), nan=-1.0), torch.nan_to_num(s.squeeze(1).float(), nan=-1.0)), "scales differ"


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (2, 129), (33, 1000), (17, 4096), (2, 14336), (3, 20001), (1, 131071)])
def test_rows_become_the_nearest_codes(dev, dtype, rows, cols):
    g = torch.Generator().manual_seed(rows * 7 + cols)
    x = torch.randn(rows, cols, generator=g)
    x[:, 0] *= 4
    check_rows(x.to(dtype), dev)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_at_the_edges_of_their_type(dev, dtype):
    fi = torch.finfo(dtype)
    g = torch.Generator().manual_seed(5)
    base = torch.randint(-254, 255, (12, 300), generator=g).double()
    base[:, 0] = 254.0                                   # quotients are whole or half: every second one a tie
    x = base.to(dtype).double()
    x[1] = 0
    x[2] *= fi.max / 254 * 0.5
    x[3] = torch.where(torch.arange(300) % 2 == 0, fi.max, -fi.max / 2)
    x[4] *= fi.tiny                                      # small normal numbers
    x[5] = torch.arange(300).double() * fi.smallest_normal * fi.eps   # subnormal ones
    x[6] = 0
    x[6, 299] = -1.0                                     # one value
    x[7, 11] = float("inf")
    x[8, 0] = float("nan")
    x[9, 150] = float("-inf")
    x[10] = fi.smallest_normal * fi.eps
    check_rows(x.to(dtype), dev)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_of_any_stride(dev, dtype):
    g = torch.Generator().manual_seed(1)
    big = torch.randn(40, 301, generator=g).to(dtype)
    for view in (big[::2], big[:, 3:200], big[1:, 1::3], big.t(), big[5:5], big[:, :0][:0]):
        if view.size(1) == 0:
            continue
        c, s, _ = oracle.codes(view)
        base = big.to(dev)
        got, scale = moe.quantize_rows(torch.as_strided(base, view.shape, view.stride(), view.storage_offset()))
        assert torch.equal(got.cpu().double(), c) and torch.equal(scale.cpu(), s.squeeze(1).float())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("E,K,N", [(1, 1, 1), (3, 70, 33), (2, 256, 512), (5, 1000, 8), (2, 17, 1030)])
@pytest.mark.parametrize("along_k", [True, False])
def test_weights_become_codes_of_their_columns(dev, dtype, E, K, N, along_k):
    g = torch.Generator().manual_seed(E + K + N)
    w = torch.randn(E, K, N, generator=g).mul_(0.02).to(dtype)
    if K > 1 and N > 2:
        w[0, :, 1] = 0
        w[E - 1, K // 2, 2] = float("inf")
    w = w.transpose(1, 2).contiguous().transpose(1, 2) if along_k else w
    c, s, _ = oracle.codes(w.permute(0, 2, 1).reshape(E * N, K))
    q, scale = moe.quantize_expert_weights(w.to(dev))
    assert torch.equal(q.cpu().double(), c.view(E, N, K).permute(0, 2, 1))
    assert torch.equal(torch.nan_to_num(scale.cpu(), nan=-1.0), torch.nan_to_num(s.view(E, N).float(), nan=-1.0))


# ---------------------------------------------------------------------------------------------------------------
# one projection
# ---------------------------------------------------------------------------------------------------------------
def weights(E, K, N, seed, layout):
    g = torch.Generator().manual_seed(seed)
    c = torch.randint(-127, 128, (E, K, N), generator=g, dtype=torch.int8)
    ws = torch.rand(E, N, generator=g) * 1e-3 + 1e-4
    if layout == "nk":
        c = c.transpose(1, 2).contiguous().transpose(1, 2)
    elif layout == "strided":                              # contiguous along neither
        c = c.permute(1, 2, 0).contiguous().permute(2, 0, 1)
    return c, ws


def linear_case(dev, dtype, T, K, N, E, k, layout="nk", gates=False, grouped_in=False, grouped_out=False, train=True, absent=(), idx=torch.int64, offsets=True,
                stride=None):
    sei, ssi, eo, gw = oracle.route(T, E, k, T + E, absent)
    w, ws = weights(E, K, N, K + N, layout)
    g = torch.Generator().manual_seed(T * 3 + K)
    x = torch.randn(T, K, generator=g).to(dtype)
    gw = gw.to(dtype) if gates else None
    rows = T if gates else T * k
    dout = torch.randn(rows, N, generator=g).to(dtype) if train else None
    # the gradient's codes: fp32 products of 2-byte values are off by three roundings, fp32 rows are taken in 64 bits
    near = 127 * 4 * 2.0 ** -24 if dtype != F32 else 127 * 2.0 ** -50
    want = oracle.linear(x, w, ws, k, sei, ssi, gw, dout, grouped_in, grouped_out, near)
    xd = x.to(dev)
    if stride:
        xd = torch.zeros(T, K + stride, dtype=dtype, device=dev)[:, 1:K + 1].copy_(xd)
    xd.requires_grad_(train)
    gd = gw.to(dev).requires_grad_(train) if gates else None
    wd = torch.empty_strided(w.shape, w.stride(), dtype=torch.int8, device=dev).copy_(w)
    assert wd.stride() == w.stride()
    y = moe.parallel_linear_int8(xd, wd, ws.to(dev), k, sei.to(dev, idx), ssi.to(dev, idx), None, eo.to(dev, idx) if offsets else None, gd, grouped_in, grouped_out)
    assert y.dtype == dtype
    h, tiny = half_step(dtype), torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    if gates:
        # fp32 rows, k products and k - 1 sums in fp32, one rounding
        close(y, want["y"], want["y_terms"] * (F32_STEPS + 2 * k * 2.0 ** -24) * 1.01 + want["y"].abs() * h * 1.01 + k * tiny, "y")
    else:
        close(y, want["y"], want["y"].abs() * (h + F32_STEPS) * 1.01 + tiny, "y")
    if not train:
        return
    y.backward(dout.to(dev))
    slack = want["dx_slack"] + want["dx_terms"] * (F32_STEPS + k * 2.0 ** -24) * 1.01 + (want["dx"].abs() + want["dx_slack"]) * h * 1.01 + k * tiny
    close(xd.grad, want["dx"], slack, "dx")
    if gates:
        assert gd.grad.dtype == dtype
        # fp32 products and sums of N terms (in any order: at most N + 1 roundings of what they come to)
        close(gd.grad, want["d_gates"], want["d_gates_terms"] * (F32_STEPS + (N + 1) * 2.0 ** -24) * 1.01 + want["d_gates"].abs() * h * 1.01 + tiny, "d_gates")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("layout", ["nk", "kn", "strided"])
@pytest.mark.parametrize("T,K,N,E,k", [(1, 64, 64, 4, 2), (5, 128, 256, 4, 2), (70, 200, 136, 3, 1), (130, 333, 77, 5, 3), (300, 512, 384, 8, 2)])
def test_linear_and_its_gradients(dev, dtype, layout, T, K, N, E, k):
    linear_case(dev, dtype, T, K, N, E, k, layout)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,K,N,E,k", [(1, 256, 128, 8, 8), (3, 64, 48, 2, 2), (257, 320, 192, 6, 2), (900, 640, 1024, 4, 3)])
def test_linear_with_gates(dev, dtype, T, K, N, E, k):
    linear_case(dev, dtype, T, K, N, E, k, "nk", gates=True)


@pytest.mark.parametrize("grouped_in,grouped_out", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("layout", ["nk", "kn"])
def test_linear_with_grouped_rows(dev, grouped_in, grouped_out, layout):
    linear_case(dev, BF16, 211, 192, 320, 5, 1 if grouped_in else 3, layout, grouped_in=grouped_in, grouped_out=grouped_out)


@pytest.mark.parametrize("K,N", [(1, 1), (1, 300), (300, 1), (15, 17), (16, 16), (127, 129), (129, 127), (1000, 1368), (2000, 33)])
@pytest.mark.parametrize("layout", ["nk", "kn"])
def test_linear_of_odd_sizes(dev, K, N, layout):
    linear_case(dev, BF16, 67, K, N, 3, 2, layout)


@pytest.mark.parametrize("T,E,absent", [(600, 1, ()), (257, 16, tuple(range(1, 15))), (40, 100, tuple(range(0, 100, 2))), (1200, 3, (0,)), (17, 70, ())])
def test_linear_of_uneven_groups(dev, T, E, absent):
    linear_case(dev, BF16, T, 256, 192, E, min(2, E - len(absent)), "nk", absent=absent)


@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
@pytest.mark.parametrize("offsets", [True, False])
def test_linear_takes_both_index_types_and_finds_its_offsets(dev, idx, offsets):
    linear_case(dev, BF16, 90, 128, 160, 7, 2, "nk", idx=idx, offsets=offsets, stride=5)


def test_linear_of_the_longest_sum(dev):
    """131071 products of +-127 * 127 in one sum: the largest magnitude that a sum can have."""
    K, N = 131071, 16
    x = torch.ones(2, K, dtype=BF16, device=dev)
    x[1] = -1
    w = torch.full((1, N, K), 127, dtype=torch.int8, device=dev)
    idx = torch.arange(2, device=dev)
    y = moe.parallel_linear_int8(x, w.transpose(1, 2), torch.full((1, N), 2.0 ** -20, device=dev), 1, torch.zeros_like(idx), idx, None, None)
    want = 127 * 127 * K * (1 / 127) * 2.0 ** -20
    assert torch.allclose(y[0].float(), torch.tensor(want, device=dev), rtol=2.0 ** -8) and torch.equal(y[0], -y[1])
    with pytest.raises(RuntimeError, match="unsupported"):
        moe.parallel_linear_int8(torch.ones(2, K + 1, dtype=BF16, device=dev), torch.ones((1, K + 1, N), dtype=torch.int8, device=dev), torch.ones((1, N), device=dev), 1,
                                 torch.zeros_like(idx), idx, None, None)


def test_linear_without_rows(dev):
    none = torch.empty(0, dtype=torch.int64, device=dev)
    x = torch.empty(0, 64, dtype=BF16, device=dev, requires_grad=True)
    w, ws = weights(4, 64, 32, 0, "nk")
    y = moe.parallel_linear_int8(x, w.to(dev), ws.to(dev), 2, none, none, None, None)
    assert y.shape == (0, 32)
    y.sum().backward()
    assert x.grad.shape == x.shape


@pytest.mark.parametrize("rows", [1, 37])
def test_rows_that_are_one_row(dev, rows):
    """Inputs and gradients whose rows are one row of memory (a stride of 0), as expand and sum().backward() make them."""
    K, N, E = 128, 96, 3
    sei, ssi, eo, _ = (t.to(dev) for t in oracle.route(rows, E, 1, 2))
    w, ws = (t.to(dev) for t in weights(E, K, N, 1, "nk"))
    one = torch.randn(K, generator=torch.Generator().manual_seed(3)).to(BF16).to(dev)
    call = lambda x: moe.parallel_linear_int8(x, w, ws, 1, sei, ssi, None, eo)   # noqa: E731
    a, b = one.expand(rows, K).requires_grad_(True), one.expand(rows, K).contiguous().requires_grad_(True)
    assert torch.equal(call(a), call(b)) and torch.equal(moe.quantize_rows(a)[0], moe.quantize_rows(b)[0])
    dout = torch.ones(N, dtype=BF16, device=dev).expand(rows, N)
    want = torch.autograd.grad(call(b), b, dout.contiguous())[0]
    assert torch.equal(torch.autograd.grad(call(a), a, dout)[0], want) and torch.equal(torch.autograd.grad(call(b).sum(), b)[0], want)
    mw = moe.Int8ExpertWeights(*(t.to(dev) for t in mlp_weights(E, K, 64, 0)))
    mlp = lambda x: moe.fused_expert_mlp_int8(x, mw, 1, ssi, eo)   # noqa: E731
    assert torch.equal(mlp(a), mlp(b))
    assert torch.equal(torch.autograd.grad(mlp(a).sum(), a)[0], torch.autograd.grad(mlp(b).sum(), b)[0])


def test_a_row_that_is_not_finite_stays_alone(dev):
    T, K, N, E, k = 40, 256, 128, 4, 2
    sei, ssi, eo, _ = oracle.route(T, E, k, 3)
    w, ws = weights(E, K, N, 1, "nk")
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(0)).to(BF16)
    args = [t.to(dev) for t in (w, ws, sei, ssi, eo)]
    good = moe.parallel_linear_int8(x.to(dev), args[0], args[1], k, args[2], args[3], None, args[4])
    x[7, 5], x[20, 0] = float("nan"), float("inf")
    bad = moe.parallel_linear_int8(x.to(dev), args[0], args[1], k, args[2], args[3], None, args[4])
    hit = torch.zeros(T, dtype=torch.bool)
    hit[[7, 20]] = True
    hit = hit.repeat_interleave(k).to(dev)
    assert torch.isnan(bad[hit]).all() and torch.equal(bad[~hit], good[~hit])


def test_the_gradient_follows_differences(dev):
    """The codes of the input are a step function; over a change that is large against a step, the difference of the outputs is the gradient's up to
    half a step per input on either side."""
    T, K, N, E = 6, 96, 80, 3
    sei, ssi, eo, _ = oracle.route(T, E, 1, 9)
    w, ws = weights(E, K, N, 4, "nk")
    g = torch.Generator().manual_seed(2)
    x, v, dout = (torch.randn(*s, generator=g, dtype=F32) for s in ((T, K), (T, K), (T, N)))
    call = lambda t: moe.parallel_linear_int8(t, w.to(dev), ws.to(dev), 1, sei.to(dev), ssi.to(dev), None, eo.to(dev))   # noqa: E731
    xd = x.to(dev).requires_grad_(True)
    call(xd).backward(dout.to(dev))
    along = float((xd.grad.double().cpu() * v.double()).sum())
    plus, minus = call((x + v).to(dev)).double().cpu(), call((x - v).to(dev)).double().cpu()
    diff = float(((plus - minus) / 2 * dout.double()).sum())
    expert = torch.empty(T, dtype=torch.int64)
    expert[ssi] = sei
    deq = w.double() * ws.double().unsqueeze(1)
    step = lambda t: t.abs().amax(1, keepdim=True).double() / 254   # noqa: E731
    push = torch.stack([(deq[expert[t]] @ dout[t].double()).abs().sum() for t in range(T)])
    gstep = torch.stack([(dout[t].double() * ws[expert[t]].double()).abs().max() / 254 * (w[expert[t]].double() * 1).abs().sum(1).mul(v[t].double().abs()).sum() for t in range(T)])
    bound = float(((step(x + v) + step(x - v)).squeeze(1) / 2 * push).sum() + gstep.sum())
    assert abs(diff - along) <= bound * 1.001, (diff, along, bound)


# ---------------------------------------------------------------------------------------------------------------
# the expert MLP
# ---------------------------------------------------------------------------------------------------------------
def mlp_weights(E, d, f, seed):
    g = torch.Generator().manual_seed(seed)
    out = []
    for over in (2, 1, 2):                                  # w1, w2, w3
        w = torch.randn(E, f, d, generator=g) * 0.05
        s = w.abs().amax(over, keepdim=True) / 127
        out += [(w / s).round().to(torch.int8), s.squeeze(over)]
    return out


def mlp_case(dev, dtype, T, d, f, E, k, gates=True, grouped_out=False, train=True, absent=()):
    sei, ssi, eo, gw = oracle.route(T, E, k, T + f, absent)
    w = mlp_weights(E, d, f, d + f)
    g = torch.Generator().manual_seed(T + d)
    x = torch.randn(T, d, generator=g).to(dtype)
    gw = gw.to(dtype) if gates else None
    dout = torch.randn(T if gates else T * k, d, generator=g).to(dtype) if train else None
    # h: 2^-24 of its segment's maximum (its 24-bit code), and the exponential's, the reciprocal's and eight fp32 roundings (2^-20 together), times 127 steps
    near = 127 * (2.0 ** -24 + 2.0 ** -20)
    want = oracle.mlp(x, w, k, sei, ssi, gw, dout, grouped_out, near)
    xd = x.to(dev).requires_grad_(train)
    gd = gw.to(dev).requires_grad_(train) if gates else None
    y = moe.fused_expert_mlp_int8(xd, moe.Int8ExpertWeights(*(t.to(dev) for t in w)), k, ssi.to(dev), eo.to(dev), gd, grouped_out)
    assert y.dtype == dtype
    h, tiny = half_step(dtype), torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    terms = want.get("y_terms", want["y"].abs())
    rounding = terms * (F32_STEPS + 2.0 ** -20 + 2 * k * 2.0 ** -24) + want["y"].abs() * h
    close(y, want["y"], want["y_slack"] * 1.01 + (rounding + want["y_slack"] * h) * 1.02 + (k + 1) * tiny, "y")
    if not train:
        return
    y.backward(dout.to(dev))
    # Gradients: one rounding to the type (half a step), and of the codes of dgate and dup, whose values are as exact as h, at most
    # 2 * 127 * 2^-18 round the other way: each moves its value by a step of at most 8 / 127 of the row's size (the largest of 2 f normal products
    # is below 12 of it for f <= 2^12, and all but 2 % of rows below 8).
    flips = (2 * 127 * 2.0 ** -18) ** 0.5 * 12 / 127
    assert norm_rel(xd.grad, want["dx"]) <= h + flips, norm_rel(xd.grad, want["dx"])
    if gates:
        assert norm_rel(gd.grad, want["d_gates"]) <= h + (2 * near) ** 0.5 * 12 / 127


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,d,f,E,k", [(1, 64, 64, 2, 1), (1, 256, 512, 8, 2), (9, 128, 192, 4, 4), (100, 320, 448, 8, 2), (515, 192, 256, 3, 2), (700, 512, 1024, 2, 1)])
def test_mlp_and_its_gradients(dev, dtype, T, d, f, E, k):
    mlp_case(dev, dtype, T, d, f, E, k)


@pytest.mark.parametrize("grouped_out", [False, True])
def test_mlp_rows_without_gates(dev, grouped_out):
    mlp_case(dev, BF16, 150, 256, 320, 5, 2, gates=False, grouped_out=grouped_out)
    mlp_case(dev, F16, 33, 128, 64, 5, 1, gates=False, grouped_out=grouped_out)


@pytest.mark.parametrize("T,E,absent", [(300, 16, tuple(range(2, 16))), (64, 80, ()), (7, 3, (1,)), (1000, 1, ())])
def test_mlp_of_uneven_groups(dev, T, E, absent):
    mlp_case(dev, BF16, T, 128, 256, E, min(2, E - len(absent)), absent=absent)


# ---------------------------------------------------------------------------------------------------------------
# sizes that take the large tiles, parts of tiles, and addresses past 32 bits
# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("layout", ["nk", "kn"])
@pytest.mark.parametrize("dtype,T,K,N,E,k,gates", [(BF16, 3000, 1088, 2304, 4, 2, True), (F32, 2100, 512, 2048, 2, 2, False), (F16, 1300, 2000, 1000, 1, 1, False),
                                                   (BF16, 40, 4096, 300, 2, 2, True), (BF16, 3, 8192, 512, 4, 1, False), (F32, 20, 5000, 130, 1, 1, False)])
def test_linear_of_many_rows_and_of_long_sums(dev, dtype, T, K, N, E, k, gates, layout):
    linear_case(dev, dtype, T, K, N, E, k, layout, gates=gates)


@pytest.mark.parametrize("T,d,f,E,k", [(2500, 512, 2048, 4, 2), (1400, 1088, 1216, 2, 1), (2, 4096, 1024, 4, 2), (30, 2048, 2112, 2, 1)])
def test_mlp_of_many_rows_and_of_long_sums(dev, T, d, f, E, k):
    mlp_case(dev, BF16, T, d, f, E, k)


def test_outputs_past_two_to_the_31_elements(dev):
    """Rows of an output of 2.3e9 elements lie where they should, at both ends."""
    T, K, N, E = 160000, 64, 14336, 2
    g = torch.Generator(device=dev).manual_seed(0)
    x = torch.randn(T, K, generator=g, device=dev).to(BF16)
    w = torch.randint(-127, 128, (E, N, K), generator=g, device=dev, dtype=torch.int8).transpose(1, 2)
    ws = torch.rand(E, N, generator=g, device=dev) * 1e-3
    idx = torch.randint(0, E, (T,), generator=g, device=dev)
    sei, ssi = idx.sort(stable=True)
    y = moe.parallel_linear_int8(x, w, ws, 1, sei, ssi, None, None)
    for t in (0, 1, 74898, 74899, 149796, T - 2, T - 1):
        c, s, _ = oracle.codes(x[t:t + 1].cpu())
        e = int(idx[t])
        want = (c @ w[e].cpu().double()) * s.float().double() * ws[e].cpu().double()
        close(y[t:t + 1], want, want.abs() * (half_step(BF16) + F32_STEPS) * 1.01 + 1e-30, f"row {t}")


# ---------------------------------------------------------------------------------------------------------------
# what does not depend on the rest of a batch, on the stream, on the call
# ---------------------------------------------------------------------------------------------------------------
def setup_mlp(dev, T, d=512, f=1024, E=8, k=2, dtype=BF16, seed=0):
    sei, ssi, eo, gw = oracle.route(T, E, k, seed)
    w = moe.Int8ExpertWeights(*(t.to(dev) for t in mlp_weights(E, d, f, seed)))
    x = torch.randn(T, d, generator=torch.Generator().manual_seed(seed)).to(dtype)
    return x.to(dev), w, ssi.to(dev), eo.to(dev), gw.to(dtype).to(dev)


def test_a_token_has_the_same_result_in_any_batch(dev):
    """Sums are exact and everything else is per row, so tiles, K parts and the other tokens change no bit."""
    T, E, k = 900, 8, 2
    x, w, ssi, eo, gates = setup_mlp(dev, T, d=1024, f=2048)
    idx = torch.empty(T * k, dtype=torch.int64, device=dev)
    idx[ssi] = torch.repeat_interleave(torch.arange(E, device=dev), torch.diff(eo, prepend=eo.new_zeros(1)))
    whole = moe.fused_expert_mlp_int8(x, w, k, ssi, eo, gates)
    for lo, hi in ((0, 1), (17, 20), (300, 364), (100, 700)):
        part = idx.view(T, k)[lo:hi].reshape(-1)
        sei, pos = part.sort(stable=True)
        offs = torch.bincount(sei, minlength=E).cumsum(0)
        got = moe.fused_expert_mlp_int8(x[lo:hi], w, k, pos, offs, gates[lo:hi])
        assert torch.equal(got, whole[lo:hi]), (lo, hi)


def mlp_step(x, w, k, ssi, eo, gates, dout):
    x, gates = x.detach().requires_grad_(True), gates.detach().requires_grad_(True)
    y = moe.fused_expert_mlp_int8(x, w, k, ssi, eo, gates)
    return [y.detach(), *torch.autograd.grad(y, (x, gates), dout)]


def test_two_streams_at_once_and_again(dev):
    cases = [setup_mlp(dev, T, seed=T) for T in (700, 3, 64, 257)]
    douts = [torch.randn_like(c[0]) for c in cases]
    want = [mlp_step(c[0], c[1], 2, *c[2:], d) for c, d in zip(cases, douts)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(2):
        got = []
        for st, c, d in zip(streams, cases, douts):
            with torch.cuda.stream(st):
                got.append(mlp_step(c[0], c[1], 2, *c[2:], d))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.parametrize("T", [1, 48, 700])
def test_calls_capture_into_graphs_that_share_the_device(dev, T):
    """Two captured calls, replayed in turn between eager ones, give the eager results bit for bit, with new inputs too."""
    x, w, ssi, eo, gates = setup_mlp(dev, T, d=1024)
    lw, ls = (t.to(dev) for t in weights(8, 1024, 520, 1, "nk"))
    sei = torch.repeat_interleave(torch.arange(8, device=dev), torch.diff(eo, prepend=eo.new_zeros(1)), output_size=ssi.numel())
    calls = [lambda: moe.fused_expert_mlp_int8(x, w, 2, ssi, eo, gates), lambda: moe.parallel_linear_int8(x, lw, ls, 2, sei, ssi, None, eo, gates)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in calls:
            c()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for c in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(c())
    for trial in range(4):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(trial)).to(x.dtype))
        for i in ((0, 1), (1, 0), (0, 0))[trial % 3]:
            graphs[i].replay()
            torch.cuda.synchronize()
            got = outs[i].clone()
            assert torch.equal(got, calls[i]()), (trial, i)


def test_a_training_step_captures_into_a_graph(dev):
    x, w, ssi, eo, gates = setup_mlp(dev, 600)
    dout = torch.randn_like(x)
    leaves = [x.requires_grad_(True), gates.requires_grad_(True)]

    def step():
        for t in leaves:
            t.grad = None
        moe.fused_expert_mlp_int8(x, w, 2, ssi, eo, gates).backward(dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    captured = [t.grad for t in leaves]
    for trial in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(trial)).to(x.dtype))
        graph.replay()
        torch.cuda.synchronize()
        got = [g.clone() for g in captured]
        step()
        assert all(torch.equal(a, t.grad) for a, t in zip(got, leaves)), trial


def test_backward_runs_again_and_for_either_input_alone(dev):
    x, w, ssi, eo, gates = setup_mlp(dev, 130)
    sei = torch.repeat_interleave(torch.arange(8, device=dev), torch.diff(eo, prepend=eo.new_zeros(1)))
    lw, ls = (t.to(dev) for t in weights(8, 512, 200, 1, "kn"))
    for call in (lambda a, b: moe.fused_expert_mlp_int8(a, w, 2, ssi, eo, b), lambda a, b: moe.parallel_linear_int8(a, lw, ls, 2, sei, ssi, None, eo, b)):
        a, b = x.detach().requires_grad_(True), gates.detach().requires_grad_(True)
        y = call(a, b)
        dout = torch.randn_like(y)
        want = torch.autograd.grad(y, (a, b), dout, retain_graph=True)
        again = torch.autograd.grad(y, (a, b), dout)
        assert all(torch.equal(u, v) for u, v in zip(want, again))
        assert torch.equal(torch.autograd.grad(call(a, gates), a, dout)[0], want[0])
        assert torch.equal(torch.autograd.grad(call(x, b), b, dout)[0], want[1])
        assert torch.equal(call(x, gates), y) and not call(x, gates).requires_grad
        # gradients that are not contiguous, or broadcast
        odd = dout.t().contiguous().t()
        assert torch.equal(torch.autograd.grad(call(a, b), a, odd)[0], want[0])
        ones = torch.autograd.grad(call(a, b).sum(), a)[0]
        assert torch.equal(ones, torch.autograd.grad(call(a, b), a, torch.ones_like(dout))[0])


def test_among_the_tools_of_autograd(dev):
    import torch.autograd.forward_ad as fwad
    from torch.utils.checkpoint import checkpoint
    x, w, ssi, eo, gates = setup_mlp(dev, 90)
    call = lambda v: moe.fused_expert_mlp_int8(v, w, 2, ssi, eo, gates)   # noqa: E731
    dout = torch.randn_like(x)

    def grad_of(f):
        v = x.detach().requires_grad_(True)
        return torch.autograd.grad(f(v), v, dout)[0] if f is call else (f(v).backward(dout), v.grad)[1]
    want = grad_of(call)
    for reentrant in (False, True):
        assert torch.equal(grad_of(lambda v: checkpoint(call, v, use_reentrant=reentrant)), want)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(dev)):
        assert torch.equal(grad_of(lambda v: call(v)), want)
    traced = torch.jit.trace(call, (x,), check_trace=False)
    other = torch.randn_like(x)
    assert torch.equal(traced(other), call(other))
    with fwad.dual_level(), pytest.raises(RuntimeError, match="(?i)jvp|forward"):
        call(fwad.make_dual(x, torch.randn_like(x)))


@pytest.mark.parametrize("gates_dtype", [F32, F16])
def test_gates_of_another_type(dev, gates_dtype):
    """Gate weights keep their own type, and so does their gradient: fp32 sums of fp32 rows, rounded once."""
    T, K, N, E, k = 120, 192, 256, 4, 2
    sei, ssi, eo, gw = oracle.route(T, E, k, 8)
    w, ws = weights(E, K, N, 2, "nk")
    g = torch.Generator().manual_seed(5)
    x, dout, gw = torch.randn(T, K, generator=g).to(BF16), torch.randn(T, N, generator=g).to(BF16), gw.to(gates_dtype)
    want = oracle.linear(x, w, ws, k, sei, ssi, gw, dout, near=127 * 5 * 2.0 ** -24)
    xd, gd = x.to(dev).requires_grad_(True), gw.to(dev).requires_grad_(True)
    y = moe.parallel_linear_int8(xd, w.to(dev), ws.to(dev), k, sei.to(dev), ssi.to(dev), None, eo.to(dev), gd)
    y.backward(dout.to(dev))
    h = half_step(BF16)
    close(y, want["y"], want["y_terms"] * (F32_STEPS + 2 * k * 2.0 ** -24) * 1.01 + want["y"].abs() * h * 1.01, "y")
    close(xd.grad, want["dx"], want["dx_slack"] * 1.01 + want["dx_terms"] * (F32_STEPS + k * 2.0 ** -24) * 1.01 + (want["dx"].abs() + want["dx_slack"]) * h * 1.01, "dx")
    assert gd.grad.dtype == gates_dtype
    close(gd.grad, want["d_gates"], want["d_gates_terms"] * (F32_STEPS + (N + 1) * 2.0 ** -24) * 1.01 + want["d_gates"].abs() * half_step(gates_dtype) * 1.01, "d_gates")


def test_mlp_without_rows(dev):
    x, w, ssi, eo, gates = setup_mlp(dev, 1)
    x0, g0 = x[:0].detach().requires_grad_(True), gates[:0].detach().requires_grad_(True)
    for grouped in (False, True):
        y = moe.fused_expert_mlp_int8(x0, w, 2, ssi[:0], torch.zeros_like(eo), None if grouped else g0, grouped)
        y.sum().backward()
        assert y.shape == (0, x.size(1)) and x0.grad.shape == x0.shape
    assert g0.grad.shape == g0.shape


def test_what_is_not_finite_reaches_its_own_rows_only(dev):
    """A weight column that is not finite reaches every row of its expert (through h), a token or a gradient row that is not only itself."""
    x, w, ssi, eo, gates = setup_mlp(dev, 60)
    dout = torch.randn_like(x)
    good = mlp_step(x, w, 2, ssi, eo, gates, dout)
    expert = torch.empty(120, dtype=torch.int64, device=dev)
    expert[ssi] = torch.repeat_interleave(torch.arange(8, device=dev), torch.diff(eo, prepend=eo.new_zeros(1)))
    bad_scale = w.w3_scale.clone()
    bad_scale[3, 100] = float("nan")
    bad = mlp_step(x, w._replace(w3_scale=bad_scale), 2, ssi, eo, gates, dout)
    hit = (expert.view(60, 2) == 3).any(1)
    for i in range(2):
        assert torch.isnan(bad[i][hit]).all() and torch.equal(bad[i][~hit], good[i][~hit])
    x2, d2 = x.clone(), dout.clone()
    x2[7, 3] = float("inf")
    d2[9] = float("-inf")
    bad = mlp_step(x2, w, 2, ssi, eo, gates, d2)
    rows = torch.arange(60, device=dev)
    assert torch.isnan(bad[0][7]).all() and torch.equal(bad[0][rows != 7], good[0][rows != 7])
    fine = (rows != 7) & (rows != 9)
    assert torch.isnan(bad[1][[7, 9]]).all() and torch.equal(bad[1][fine], good[1][fine])


# ---------------------------------------------------------------------------------------------------------------
# the block and the layer
# ---------------------------------------------------------------------------------------------------------------
def make_block(dev, dtype=BF16, d=256, f=512, E=8, **kw):
    torch.manual_seed(0)
    return moe.ScatterMoEBlock(d, f, E, dtype=dtype, device=dev, **kw)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_quantised_block_is_the_operators_one_after_the_other(dev, dtype):
    block = make_block(dev, dtype)
    stored = {n: getattr(block, n).detach().clone().view(8, 512, 256) for n in ("w1", "w2", "w3")}
    assert block.quantize_experts() is block and block.is_quantized and block.quantize_experts() is block
    assert sorted(n for n, _ in block.named_parameters()) == ["router"]
    weights_ = moe.Int8ExpertWeights.quantize(stored["w1"], stored["w2"], stored["w3"])
    for n, t in weights_._asdict().items():
        assert torch.equal(getattr(block, n), t), n
    x = torch.randn(3, 50, 256, device=dev).to(dtype)
    with torch.no_grad():
        hidden, none = block(x)
        flat = x.view(-1, 256)
        out, ew, ei = moe.moe_layer_forward_int8(flat, block.router, weights_)
        assert none is None and torch.equal(hidden.view(-1, 256), out)
        _, rw, ri = moe.forward_router(flat, block.router, 2)
        assert torch.equal(ei.long(), ri) and torch.equal(ew, rw)
        sei, ssi = moe.flatten_and_sort(ri, 8)
        eo = torch.bincount(sei, minlength=8).cumsum(0)
        assert torch.equal(moe.fused_expert_mlp_int8(flat, weights_, 2, ssi, eo, rw), out)
        # three projections and torch's SwiGLU: the same up to the fp32 roundings of h, which a code or two may show
        g1, u1 = (moe.parallel_linear_int8(flat.float(), getattr(weights_, n).transpose(1, 2), getattr(weights_, n + "_scale"), 2, sei, ssi, None, eo, grouped_out=True)
                  for n in ("w1", "w3"))
        h = torch.nn.functional.silu(g1) * u1
        y = moe.parallel_linear_int8(h, weights_.w2, weights_.w2_scale, 1, sei, ssi, None, eo, gates=None, grouped_in=True)
        ref = (y.view(-1, 2, 256) * rw.unsqueeze(-1)).sum(1)
        assert norm_rel(out, ref.double().cpu()) <= half_step(dtype) + (2 * 127 * 2.0 ** -19) ** 0.5 * 12 / 127


def test_a_quantised_block_learns_what_lies_around_it(dev):
    """Gradients of the hidden states and the router against those of the definition's parts: experts by the oracle, the router by autograd."""
    block = make_block(dev).quantize_experts()
    x = torch.randn(70, 256, device=dev).to(BF16).requires_grad_(True)
    dout = torch.randn(70, 256, device=dev).to(BF16)
    block(x)[0].backward(dout)
    xr = x.detach().cpu().double().requires_grad_(True)
    wr = block.router.detach().cpu().double().requires_grad_(True)
    w, idx = torch.softmax(xr @ wr.t(), -1).topk(2, -1)
    w = w / w.sum(-1, keepdim=True)
    sei, ssi = idx.reshape(-1).sort(stable=True)
    parts = [getattr(block, n).cpu() for n in moe.Int8ExpertWeights._fields]
    want = oracle.mlp(x.detach().cpu(), parts, 2, sei, ssi, w.detach(), dout.cpu())
    (w * want["d_gates"]).sum().backward()
    flips = (2 * 127 * 2.0 ** -18) ** 0.5 * 12 / 127
    assert norm_rel(x.grad, want["dx"] + xr.grad) <= 2 * half_step(BF16) + flips     # (two gradients, each rounded, and their sum)
    # weights of the router come from fp32 logits of bf16 values: 2^-20 of the largest; d_gates carries the flips of h
    assert norm_rel(block.router.grad, wr.grad) <= half_step(BF16) + 2 * flips


def test_a_quantised_block_loads_what_it_saved(dev):
    a, b = make_block(dev).quantize_experts(), make_block(dev, E=8).quantize_experts()
    with torch.no_grad():
        b.router.zero_()
        b.w1.zero_()
    b.load_state_dict(a.state_dict())
    x = torch.randn(9, 256, device=dev).to(BF16)
    with torch.no_grad():
        assert torch.equal(a(x)[0], b(x)[0])
        empty, _ = a(x[:0])
        assert empty.shape == (0, 256)
        biased = make_block(dev, bias=True, return_bias=True).quantize_experts()
        out, bias = biased(x)
        assert bias is biased.bias and out.shape == x.shape
    with pytest.raises(ValueError, match="adapters"):
        make_block(dev, lora_r=16).quantize_experts()
    with pytest.raises((RuntimeError, TypeError), match="float32"):
        a.to(BF16)(x)                                          # its scales would be bf16


def test_adapters_beside_quantised_weights(dev):
    """A frozen projection in 8 bits and a trained low-rank one beside it: the sum of two calls, with the gradients of both."""
    T, K, N, E, k, r = 300, 256, 384, 4, 2, 16
    sei, ssi, eo, gates = (t.to(dev) for t in oracle.route(T, E, k, 1))
    w, ws = (t.to(dev) for t in weights(E, K, N, 3, "nk"))
    g = torch.Generator().manual_seed(4)
    mk = lambda *s: (torch.randn(*s, generator=g) * 0.1).to(BF16).to(dev).requires_grad_(True)   # noqa: E731
    x, a, b, dout = mk(T, K), mk(E, K, r), mk(E, r, N), mk(T * k, N).detach()
    base = moe.parallel_linear_int8(x, w, ws, k, sei, ssi, None, eo)
    low = moe.parallel_linear(moe.parallel_linear(x, a, k, sei, ssi, None, eo, grouped_out=True), b, 1, sei, ssi, None, eo, grouped_in=True)
    (base + low).backward(dout)
    parts = [torch.autograd.grad(moe.parallel_linear_int8(x, w, ws, k, sei, ssi, None, eo), x, dout)[0]]
    low = moe.parallel_linear(moe.parallel_linear(x, a, k, sei, ssi, None, eo, grouped_out=True), b, 1, sei, ssi, None, eo, grouped_in=True)
    parts += torch.autograd.grad(low, (x, a, b), dout)
    assert torch.equal(x.grad, parts[0] + parts[1]) and torch.equal(a.grad, parts[2]) and torch.equal(b.grad, parts[3])
