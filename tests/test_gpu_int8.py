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
        # rows rounded to the type, then (k products and k - 1 sums in fp32) and rounded again
        close(y, want["y"], want["y_terms"] * (h + F32_STEPS + 2 * k * 2.0 ** -24) * 1.01 + want["y"].abs() * h * 1.01 + k * tiny, "y")
    else:
        close(y, want["y"], want["y"].abs() * (h + F32_STEPS) * 1.01 + tiny, "y")
    if not train:
        return
    y.backward(dout.to(dev))
    slack = want["dx_slack"] + want["dx_terms"] * ((h if k > 1 else 0.0) + F32_STEPS + k * 2.0 ** -24) * 1.01 + (want["dx"].abs() + want["dx_slack"]) * h * 1.01 + k * tiny
    close(xd.grad, want["dx"], slack, "dx")
    if gates:
        assert gd.grad.dtype == dtype
        # fp32 products and sums of N terms (in any order: at most N + 1 roundings of what they come to)
        close(gd.grad, want["d_gates"], want["d_gates_terms"] * (h + F32_STEPS + (N + 1) * 2.0 ** -24) * 1.01 + want["d_gates"].abs() * h * 1.01 + tiny, "d_gates")


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
    rounding = terms * ((h if gates else 0.0) + F32_STEPS + 2.0 ** -20 + 2 * k * 2.0 ** -24) + want["y"].abs() * h
    close(y, want["y"], want["y_slack"] * 1.01 + (rounding + want["y_slack"] * h) * 1.02 + (k + 1) * tiny, "y")
    if not train:
        return
    y.backward(dout.to(dev))
    # Gradients: rows rounded to the type (half a step) and summed (half a step), and of the codes of dgate and dup, whose values are as exact as h, at most
    # 2 * 127 * 2^-18 round the other way: each moves its value by a step of at most 8 / 127 of the row's size (the largest of 2 f normal products
    # is below 12 of it for f <= 2^12, and all but 2 % of rows below 8).
    flips = (2 * 127 * 2.0 ** -18) ** 0.5 * 12 / 127
    assert norm_rel(xd.grad, want["dx"]) <= 2 * h + flips, norm_rel(xd.grad, want["dx"])
    if gates:
        assert norm_rel(gd.grad, want["d_gates"]) <= 2 * h + (2 * near) ** 0.5 * 12 / 127


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
