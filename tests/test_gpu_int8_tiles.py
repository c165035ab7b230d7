"""Expert products over 8-bit weights, tile by tile: every case names the tile size and the K parts that its products take, and the groups' sizes decide how full the tiles are
and how many parts the device cuts them into.  Results are compared element by element with the definition in 64 bits."""
import ctypes

import pytest
import torch

import moe_distributed_training_amd as moe
from moe_distributed_training_amd._lib import lib
from oracle import int8_oracle as oracle
from test_gpu_int8_edges import close, mlp_weights

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
MIN_PART = 4          # K tiles of 128 that a part has at least


def plan(R, E, K, N, pair=False, nseg=1):
    parts = ctypes.c_int(0)
    return lib.moe_int8_debug_tile(R, E, K, N, int(pair), nseg, ctypes.addressof(parts)), parts.value


def cut(counts, K, N, pair=False, nseg=1):
    """(tile, K parts of the tiles of the last round) of a launch over groups of these sizes, as the device cuts them."""
    tile, most = plan(sum(counts), len(counts), K, N, pair, nseg)
    cols = tile // 2 if pair else tile
    tiles, ktiles = sum(-(-c // tile) for c in counts) * -(-N // cols), -(-K // 128) * nseg
    places = torch.cuda.get_device_properties(0).multi_processor_count // 8 * 8 * (256 // tile)
    left, parts = tiles % places, 1
    while parts * 2 <= most and left * parts * 2 <= places and ktiles // (parts * 2) >= MIN_PART:
        parts *= 2
    return (tile, parts) if left else (tile, 1)


def grouped(counts, seed):
    """One expert per row, groups of these sizes, rows of a group anywhere in the batch."""
    sei = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
    return sei, torch.randperm(sum(counts), generator=torch.Generator().manual_seed(seed)), torch.tensor(counts).cumsum(0)


# groups that fill a tile of 256 in every way: its 16-row blocks are dealt to two rows of waves, which run one of several copies of the loop
UNEVEN = [1, 15, 16, 17, 33, 64, 100, 128, 129, 160, 200, 240, 256, 257, 300, 511]
FULL_CHIP = [700, 600, 520, 400, 300, 260, 130, 90]       # 17 row tiles of 256: with 16 column tiles one round of 256 compute units and 16 tiles more


# ---------------------------------------------------------------------------------------------------------------
# one projection
# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("layout", ["nk", "kn"])
@pytest.mark.parametrize("dtype,counts,K,N,forward,backward", [
    (BF16, UNEVEN, 1088, 2304, (256, 1), (128, 1)), (F16, UNEVEN, 512, 4096, (256, 1), (128, 1)), (F32, UNEVEN, 1000, 4104, (256, 1), (128, 1)),
    (BF16, [150, 150], 4096, 512, (256, 8), (128, 1)), (F32, [190, 110], 4000, 520, (256, 8), (128, 1)), (BF16, [200], 4096, 1024, (256, 8), (128, 1)),
    (F16, [0, 77, 223, 0], 4096, 1000, (256, 4), (128, 1)), (BF16, FULL_CHIP, 4096, 4096, (256, 2), (256, 2)),
    (BF16, [48], 4096, 512, (128, 8), (128, 1)), (F32, [3, 0, 60, 1], 8192, 300, (128, 8), (128, 1))])
def test_linear(dev, dtype, counts, K, N, forward, backward, layout):
    assert cut(counts, K, N) == forward and cut(counts, N, K) == backward
    T, E = sum(counts), len(counts)
    sei, ssi, eo = grouped(counts, K)
    g = torch.Generator().manual_seed(N)
    w = torch.randint(-127, 128, (E, N, K) if layout == "nk" else (E, K, N), generator=g, dtype=torch.int8)
    ws = torch.rand(E, N, generator=g) * 1e-3 + 1e-4
    x, dout = torch.randn(T, K, generator=g).to(dtype), torch.randn(T, N, generator=g).to(dtype)
    wk = w.transpose(1, 2) if layout == "nk" else w
    want = oracle.linear(x, wk, ws, 1, sei, ssi, None, dout, near=127 * 2.0 ** -29)
    pad = (lambda t: t) if w.size(2) % 16 == 0 else (lambda t: torch.nn.functional.pad(t, (0, -t.size(2) % 16))[:, :, :t.size(2)])   # 16-byte rows: read in place
    wd = pad(w.to(dev))
    xd = x.to(dev).requires_grad_(True)
    y = moe.parallel_linear_int8(xd, wd.transpose(1, 2) if layout == "nk" else wd, ws.to(dev), 1, sei.to(dev), ssi.to(dev), None, eo.to(dev))
    close(y, want["y"], want["y"].abs() * 6 * 2.0 ** -24, dtype, "y")
    close(torch.autograd.grad(y, xd, dout.to(dev))[0], want["dx"], want["dx_slack"] + want["dx_terms"] * 6 * 2.0 ** -24, dtype, "dx")


# ---------------------------------------------------------------------------------------------------------------
# the expert MLP
# ---------------------------------------------------------------------------------------------------------------
# groups, d, f, and what the products of gate and up, of h, of dh and of dx take
MLP = [
    (UNEVEN, 512, 4096, (256, 1), (128, 1), (256, 1), (256, 4)),
    ([1100], 512, 4096, (256, 1), (128, 1), (128, 1), (256, 8)),
    ([600, 500], 512, 4160, (256, 1), (128, 1), (128, 1), (256, 8)),
    ([1, 500, 400, 899], 512, 8192, (256, 1), (256, 4), (256, 1), (256, 8)),
    ([170, 130], 4096, 256, (256, 8), (128, 1), (128, 4), (128, 1)),
    ([299, 1], 4096, 512, (256, 8), (128, 1), (256, 8), (128, 1)),
    ([200], 1024, 4096, (128, 1), (256, 8), (128, 1), (256, 8)),
    ([1500, 600], 4096, 64, (256, 8), (256, 1), (128, 4), (256, 1)),
    ([5, 40], 2048, 2112, (128, 1), (128, 1), (128, 1), (128, 4)),
]


def mlp_inputs(dtype, counts, d, f):
    sei, ssi, eo = grouped(counts, d + f)
    g = torch.Generator().manual_seed(f)
    T = sum(counts)
    x, dout = torch.randn(T, d, generator=g).to(dtype), torch.randn(T, d, generator=g).to(dtype)
    return x, dout, mlp_weights(len(counts), d, f, d), sei, ssi, eo, (torch.rand(T, 1, generator=g) + 0.25).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", MLP, ids=lambda c: f"{sum(c[0])}-{c[1]}-{c[2]}")
def test_mlp(dev, dtype, case):
    counts, d, f = case[:3]
    assert (cut(counts, d, f, pair=True), cut(counts, f, d), cut(counts, d, f), cut(counts, f, d, nseg=2)) == case[3:]
    x, dout, w, sei, ssi, eo, gates = mlp_inputs(dtype, counts, d, f)
    want = oracle.mlp_bounds(x, w, 1, sei, ssi, gates, dout)
    wd = moe.Int8ExpertWeights(*(t.to(dev) for t in w))
    xd, gd = x.to(dev).requires_grad_(True), gates.to(dev).requires_grad_(True)
    y = moe.fused_expert_mlp_int8(xd, wd, 1, ssi.to(dev), eo.to(dev), gd)
    got = torch.autograd.grad(y, (xd, gd), dout.to(dev))
    close(y, want["y"], want["y_slack"], dtype, "y")
    close(got[0], want["dx"], want["dx_slack"], dtype, "dx")
    close(got[1], want["d_gates"], want["d_gates_slack"], dtype, "d_gates")
    with torch.no_grad():                                  # gate and up not stored: the same h
        assert torch.equal(moe.fused_expert_mlp_int8(xd, wd, 1, ssi.to(dev), eo.to(dev), gd), y)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,d,f,E,k", [(1, 256, 512, 8, 2), (70, 320, 448, 8, 2), (333, 512, 1088, 4, 3), (700, 192, 256, 3, 2)])
def test_mlp_gradients_element_by_element(dev, dtype, T, d, f, E, k):
    """Top-k routing: dx is a sum over a token's experts."""
    sei, ssi, eo, gates = oracle.route(T, E, k, T)
    g = torch.Generator().manual_seed(d)
    x, dout, gates = torch.randn(T, d, generator=g).to(dtype), torch.randn(T, d, generator=g).to(dtype), gates.to(dtype)
    w = mlp_weights(E, d, f, 3)
    want = oracle.mlp_bounds(x, w, k, sei, ssi, gates, dout)
    xd, gd = x.to(dev).requires_grad_(True), gates.to(dev).requires_grad_(True)
    y = moe.fused_expert_mlp_int8(xd, moe.Int8ExpertWeights(*(t.to(dev) for t in w)), k, ssi.to(dev), eo.to(dev), gd)
    got = torch.autograd.grad(y, (xd, gd), dout.to(dev))
    close(y, want["y"], want["y_slack"], dtype, "y")
    close(got[0], want["dx"], want["dx_slack"], dtype, "dx")
    close(got[1], want["d_gates"], want["d_gates_slack"], dtype, "d_gates")


# ---------------------------------------------------------------------------------------------------------------
# parts that meet: again, on several streams at once, in graphs
# ---------------------------------------------------------------------------------------------------------------
MEETING = [MLP[0], MLP[1], MLP[3], MLP[4], MLP[5], MLP[8]]      # parts of either tile size in every product


def step(a):
    x, w, ssi, eo, gates, dout = a
    x, gates = x.detach().requires_grad_(True), gates.detach().requires_grad_(True)
    y = moe.fused_expert_mlp_int8(x, w, 1, ssi, eo, gates)
    return [y.detach(), *torch.autograd.grad(y, (x, gates), dout)]


def on_device(dev, case):
    x, dout, w, sei, ssi, eo, gates = mlp_inputs(BF16, *case[:3])
    return x.to(dev), moe.Int8ExpertWeights(*(t.to(dev) for t in w)), ssi.to(dev), eo.to(dev), gates.to(dev), dout.to(dev)


def test_parts_on_several_streams_at_once_and_again(dev):
    args = [on_device(dev, c) for c in MEETING]
    want = [step(a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    for _ in range(3):
        got = []
        for st, a in zip(streams, args):
            with torch.cuda.stream(st):
                got.append(step(a))
        torch.cuda.synchronize()
        for u, v in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(u, v))


@pytest.mark.parametrize("first,second", [(0, 3), (1, 4), (2, 5)])
def test_parts_in_graphs_replayed_in_turn(dev, first, second):
    """Forward and backward of two captured steps, replayed in turn and between eager calls, with new inputs each time."""
    args = [on_device(dev, MEETING[i]) for i in (first, second)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a in args:
            step(a)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for a in args:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(a))
    for trial in range(4):
        for a in args:
            a[0].copy_(torch.randn(a[0].shape, generator=torch.Generator().manual_seed(trial)).to(BF16))
        for i in ((0, 1), (1, 0), (0, 0, 1))[trial % 3]:
            graphs[i].replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in outs[i]]
            assert all(torch.equal(u, v) for u, v in zip(got, step(args[i]))), (trial, i)
