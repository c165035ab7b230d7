"""The SwiGLU that keeps its inputs in 8 bits against its definition in 64 bits.

Codes are those of the exact quotients, so a gradient is off by its last rounding, by the rounding of the scales (2^-24 each) and by those of the formula in fp32: the
exponential and the reciprocal of a 16-bit type are the hardware's, each within 2^-22, and an argument's rounding costs |x| 2^-24 of the exponential
(|g| (1 - s) <= 1.3 |g s|-wise bounded: at most 12 of 2^-24 where the sigmoid's complement matters)."""
import pytest
import torch

import moe_distributed_training_amd as moe
from moe_distributed_training_amd import _lib
from oracle import fp4_oracle as oracle

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def close(got, want, slack, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    both = torch.isnan(want)
    assert torch.equal(torch.isnan(got), both), f"{what}: NaN elsewhere than expected"
    over = torch.where(both | (got == want), torch.full_like(want, -1.0), (got - want).abs() - slack)   # (infinities are equal, or as far off as can be)
    assert over.numel() == 0 or float(over.max()) <= 0, f"{what}: {float(over.max()):.3g} past its bound at {torch.nonzero(over == over.max())[0].tolist()}"


def bound(v, terms, x, dtype, factor):
    # (the relative error of exp(-x) is (|x| + 4) 2^-24 at most; it reaches the sigmoid times its complement, which falls as exp(-|x|) where x > 0)
    fi = torch.finfo(dtype)
    rel = (24 + x.abs()) * 2.0 ** -24
    # A sigmoid below 2^-126 = 1 / (1 + exp(-x)) has a denominator above 2^126, whose reciprocal is no normal number (from 2^128 on it is an infinity's): zero may
    # stand for it, at a cost of 2^-126 times what it is multiplied by.
    return fi.eps / 2 * v.abs() + rel * terms * (1 + fi.eps) + fi.smallest_normal * fi.eps + 2.0 ** -126 * factor


def check(dev, gate, up, dh, move=lambda t: t):
    dtype = gate.dtype
    h, dg, du, dgt, dut = oracle.swiglu(gate, up, dh)
    a, b = (move(t.to(dev)).detach().requires_grad_(True) for t in (gate, up))
    y = moe.swiglu_8bit(a, b)
    assert y.dtype == dtype and y.is_contiguous()
    close(y, h, bound(h, h.abs(), gate.double(), dtype, (gate.double() * up.double()).abs()), "h")
    with torch.no_grad():
        assert torch.equal(moe.swiglu_8bit(a, b).nan_to_num(nan=-9.0), y.nan_to_num(nan=-9.0))
    ga, gb = torch.autograd.grad(y, [a, b], move(dh.to(dev)))
    g8, u8, d = oracle.kept(gate)[0], oracle.kept(up)[0], dh.double()
    close(ga, dg, bound(dg, dgt, g8, dtype, (d * u8).abs() * (1 + g8.abs())), "dgate")
    close(gb, du, bound(du, dut, g8, dtype, (d * g8).abs()), "dup")


def draw(rows, cols, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    size = torch.exp(0.5 * torch.randn(rows, 1, generator=g))
    return tuple((s * torch.randn(rows, cols, generator=g)).to(dtype) for s in (2 * size, size, torch.ones(1)))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 63), (2, 64), (5, 65), (17, 200), (33, 1368), (64, 1355), (300, 512), (1, 14336), (1000, 24)])
def test_against_64_bits(dev, dtype, rows, cols):
    check(dev, *draw(rows, cols, dtype, rows + cols))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_halves_of_a_joint_matrix_and_other_strides(dev, dtype):
    gate, up, dh = draw(37, 192, dtype, 4)
    check(dev, gate, up, dh, lambda t: torch.cat((t, t), 1)[:, :192])
    check(dev, gate, up, dh, lambda t: torch.cat((t, t), 1)[:, 192:])
    check(dev, gate, up, dh, lambda t: t.t().contiguous().t())
    check(dev, gate, up, dh, lambda t: torch.cat((t[:, :1], t), 1)[:, 1:])    # unaligned rows


def test_more_dimensions(dev):
    gate, up, dh = (t.view(3, 4, 128).to(dev) for t in draw(12, 128, BF16, 2))
    a, b = gate.clone().requires_grad_(True), up.clone().requires_grad_(True)
    y = moe.swiglu_8bit(a, b)
    y.backward(dh)
    a2, b2 = gate.view(12, 128).clone().requires_grad_(True), up.view(12, 128).clone().requires_grad_(True)
    y2 = moe.swiglu_8bit(a2, b2)
    y2.backward(dh.view(12, 128))
    assert y.shape == (3, 4, 128) and torch.equal(y.view(12, 128), y2) and torch.equal(a.grad.view(12, 128), a2.grad) and torch.equal(b.grad.view(12, 128), b2.grad)
    v = moe.swiglu_8bit(gate[0, 0], up[0, 0])
    assert torch.equal(v, y2[0])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_codes_at_borders(dev, dtype):
    """Quotients that are whole or half: every second one a tie, which goes to the even code."""
    g = torch.Generator().manual_seed(8)
    v = torch.randint(-254, 255, (40, 128), generator=g).double()
    v[:, 0] = v[:, 64] = 254.0
    gate = (v / 64).to(dtype)
    up = v.flip(0).to(dtype)
    up[:, 0] = up[:, 64] = 254.0
    check(dev, gate, up, torch.ones(40, 128).to(dtype))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_what_is_not_finite_stays_in_its_block(dev, dtype):
    gate, up, dh = draw(6, 200, dtype, 3)
    gate[1, 70], up[3, 5], gate[4, 199] = float("nan"), float("inf"), float("-inf")
    gate[0, :64] = 0
    up[2, 64:128] = 0
    check(dev, gate, up, dh)


def test_large_arguments(dev):
    for dtype in (BF16, F16, F32):
        gate = torch.linspace(-300, 300, 640).view(2, 320).to(dtype)
        check(dev, gate, torch.ones(2, 320).to(dtype), torch.ones(2, 320).to(dtype))


def test_gradient_against_differences(dev):
    """Where the codes hold the inputs exactly (whole numbers of steps of a block), the gradient is that of h."""
    g = torch.Generator().manual_seed(1)
    q = torch.randint(-127, 128, (8, 64), generator=g).double()
    q[:, 0] = 127
    gate, up = (q / 32).float(), (q.flip(1).clone().index_fill_(1, torch.tensor([3]), 127) / 64).float()
    a, b = gate.to(dev).requires_grad_(True), up.to(dev).requires_grad_(True)
    ga, gb = torch.autograd.grad(moe.swiglu_8bit(a, b).sum(), [a, b])
    f = lambda x, y: x * torch.sigmoid(x) * y
    e = 1e-4
    da = (f(gate.double() + e, up.double()) - f(gate.double() - e, up.double())) / (2 * e)
    db = (f(gate.double(), up.double() + e) - f(gate.double(), up.double() - e)) / (2 * e)
    # differences: third derivative times e^2 / 6 (below 1 * up) and 64-bit cancellation; gradients: fp32
    assert float((ga.double().cpu() - da).abs().max()) < 4e-6 and float((gb.double().cpu() - db).abs().max()) < 4e-6


def test_empty(dev):
    for shape in ((0, 64), (3, 0), (0,)):
        a = torch.empty(shape, device=dev, requires_grad=True)
        b = torch.empty(shape, device=dev, requires_grad=True)
        y = moe.swiglu_8bit(a, b)
        assert y.shape == shape
        ga, gb = torch.autograd.grad(y.sum(), [a, b])
        assert ga.shape == shape and gb.shape == shape


def test_what_is_kept_is_small(dev):
    rows, cols = 512, 4096
    gate, up = (torch.randn(rows, cols, device=dev, dtype=BF16, requires_grad=True) for _ in range(2))
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = moe.swiglu_8bit(gate, up)
    held = torch.cuda.memory_allocated() - before - y.numel() * 2
    assert held <= 2 * rows * cols * 1.0625 + 4096
    assert _lib.lib.moe_swiglu8_kept_bytes(rows, cols) <= 2 * rows * cols * 1.0625 + 1024


def test_backward_again_alone_and_through_hooks(dev):
    gate, up, dh = (t.to(dev) for t in draw(40, 200, BF16, 5))
    a, b = gate.requires_grad_(True), up.requires_grad_(True)
    y = moe.swiglu_8bit(a, b)
    want = torch.autograd.grad(y, (a, b), dh, retain_graph=True)
    assert all(torch.equal(u, v) for u, v in zip(torch.autograd.grad(y, (a, b), dh), want))
    for i, (u, v) in enumerate(((a, b.detach()), (a.detach(), b))):
        assert torch.equal(torch.autograd.grad(moe.swiglu_8bit(u, v), (a, b)[i], dh)[0], want[i])
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: torch.stack((t, t), -1).to(dev)[..., 0]):
        y = moe.swiglu_8bit(a, b)
    assert all(torch.equal(u, v) for u, v in zip(torch.autograd.grad(y, (a, b), dh), want))
    # one tensor twice, and a gradient without strides
    y = moe.swiglu_8bit(a, a)
    ga, = torch.autograd.grad(y, a, torch.ones((), dtype=BF16, device=dev).expand(40, 200))
    one = torch.autograd.grad(moe.swiglu_8bit(a, gate.detach().clone().requires_grad_(True)), a, torch.ones_like(y))[0]
    two = torch.autograd.grad(moe.swiglu_8bit(a.detach(), a), a, torch.ones_like(y))[0]
    assert torch.equal(ga, one + two)


def test_steps_in_graphs_between_eager_ones_and_on_two_streams(dev):
    sets = [[t.to(dev) for t in draw(*s, BF16, 7)] for s in ((300, 512), (33, 200))]
    leaves = [[t.requires_grad_(True) for t in s[:2]] for s in sets]

    def step(i):
        for t in leaves[i]:
            t.grad = None
        moe.swiglu_8bit(*leaves[i]).backward(sets[i][2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in (0, 1, 0, 1):
            step(i)
    torch.cuda.current_stream().wait_stream(side)
    graphs, grads, pool = [], [], None
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=pool):
            step(i)
        pool = pool or graphs[0].pool()
        grads.append([t.grad for t in leaves[i]])
    for trial, i in enumerate((0, 1, 1, 0, 0)):
        with torch.no_grad():
            leaves[i][0].copy_(torch.randn(leaves[i][0].shape, generator=torch.Generator().manual_seed(trial)).to(BF16))
        graphs[i].replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in grads[i]]
        step(i)
        assert all(torch.equal(u, t.grad) for u, t in zip(got, leaves[i])), trial
    want = [[t.grad.clone() for t in leaves[i]] for i in range(2) if step(i) is None]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            got.append(torch.autograd.grad(moe.swiglu_8bit(*leaves[i]), leaves[i], sets[i][2]))
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for g, w in zip(got, want) for u, v in zip(g, w))


def test_more_values_than_32_bits_count(dev):
    rows, cols = 160000, 14336
    gate, up, dh = (torch.empty(rows, cols, dtype=BF16, device=dev).normal_() for _ in range(3))
    a, b = gate.requires_grad_(True), up.requires_grad_(True)
    y = moe.swiglu_8bit(a, b)
    ga, gb = torch.autograd.grad(y, (a, b), dh)
    for part in (slice(0, 9), slice(149795, 149805), slice(rows - 9, rows)):   # (2^31 lies in row 149796)
        u, v = (t[part].detach().clone().requires_grad_(True) for t in (gate, up))
        z = moe.swiglu_8bit(u, v)
        assert torch.equal(y[part], z)
        assert all(torch.equal(p, q) for p, q in zip((ga[part], gb[part]), torch.autograd.grad(z, (u, v), dh[part])))
