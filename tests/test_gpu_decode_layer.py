"""The layer for a few tokens, over 16-bit and 4-bit weights, against its definition in 64 bits.

What an output element may be off by: its own last rounding; the roundings of 32-bit sums over d and f (in units of the sums of their terms' magnitudes, those of gate and up
carried through SwiGLU and the down projection); the two numbers of the type that h travels as (bf16: 2^-17 of it, fp16: 2^-23, or half a subnormal step); the hardware exponential's and
the weights' few 2^-24."""
import pytest
import torch

import moe_distributed_training_amd as moe
from oracle import fp4_oracle as oracle

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def make(T, d, f, E, k, dtype, bits, seed=0):
    g = torch.Generator().manual_seed(seed * 31 + T + d + f + E)
    x = (torch.randn(T, d, generator=g) * torch.exp(0.4 * torch.randn(T, 1, generator=g))).to(dtype)
    wg = (torch.randn(E, d, generator=g) * 0.05).to(dtype)
    w = [torch.randn(E, f, d, generator=g) * 0.05 for _ in range(3)]
    if bits == 16:
        w = [t.to(dtype) for t in w]
        return x, wg, w, (w[0].double(), w[2].double(), w[1].double().transpose(1, 2))
    q = [oracle.quantize(w[0].transpose(1, 2)), oracle.quantize(w[1]), oracle.quantize(w[2].transpose(1, 2))]
    return x, wg, q, (oracle.weights(*q[0], d), oracle.weights(*q[2], d), oracle.weights(*q[1], f))


def run(dev, x, wg, w, k, normalize=True, bits=16):
    with torch.no_grad():
        if bits == 16:
            return moe.moe_layer_decode(x.to(dev), wg.to(dev), *(t.to(dev) for t in w), k, normalize)
        weights = moe.Fp4ExpertWeights(*(t.to(dev) for q in w for t in q))
        return moe.moe_layer_forward_fp4(x.to(dev), wg.to(dev), weights, k, normalize)


def slack_of(out, terms, back, w2_sum, d, f, dtype):
    a = 2.0 ** -24
    h = 2.0 ** -17 if dtype == BF16 else 2.0 ** -22
    return (torch.finfo(dtype).eps / 2 * out.abs() + (d + 24) * a * back + ((f + 64) * a + h) * terms + 2.0 ** -24 * w2_sum * (dtype == F16)) * 1.01


def check(dev, T, d, f, E, k, dtype, bits, normalize=True, seed=0):
    x, wg, w, (w1, w3, w2) = make(T, d, f, E, k, dtype, bits, seed)
    want, weights, idx, terms, back = oracle.layer(x, wg, w1, w3, w2, k, normalize)
    out, ew, ei = run(dev, x, wg, w, k, normalize, bits)
    assert out.dtype == dtype and out.shape == (T, d) and ew.dtype == torch.float32 and ei.dtype == torch.int32
    assert torch.equal(ei.cpu().long(), idx), "choices differ"
    # logits are off by (d + 8) 2^-24 of their terms, weights by twice that
    lt = (x.double().abs() @ wg.double().abs().t()).amax()
    assert float(((ew.double().cpu() - weights) / weights).abs().max()) <= 2 * ((d + 8) * lt + 16) * 2.0 ** -24
    w2_sum = sum((w2[idx[:, j]].abs().sum(-1) * weights[:, j, None]) for j in range(k))
    over = (out.double().cpu() - want).abs() - slack_of(want, terms + 0, back, w2_sum, d, f, dtype) - 2 * ((d + 8) * lt + 16) * 2.0 ** -24 * terms
    assert float(over.max()) <= 0, f"{float(over.max()):.3g} past its bound at {torch.nonzero(over == over.max())[0].tolist()}"
    return out, ew, ei


SIZES = [  # T, d, f, E, k
    (1, 64, 64, 1, 1), (1, 128, 64, 8, 2), (2, 64, 192, 4, 2), (3, 256, 512, 8, 2), (16, 128, 128, 2, 1), (7, 192, 320, 16, 4), (16, 256, 64, 64, 8), (5, 320, 128, 96, 3),
    (16, 64, 64, 256, 16), (13, 1024, 256, 8, 2), (9, 448, 960, 3, 3), (4, 2176, 1088, 4, 2), (16, 64, 64, 1, 1),
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,d,f,E,k", SIZES)
def test_layer(dev, T, d, f, E, k, dtype, bits):
    check(dev, T, d, f, E, k, dtype, bits)


@pytest.mark.parametrize("bits", [16, 4])
def test_weights_that_are_not_normalised(dev, bits):
    check(dev, 6, 128, 192, 8, 3, BF16, bits, normalize=False)


@pytest.mark.parametrize("bits", [16, 4])
def test_every_number_of_tokens(dev, bits):
    for T in range(1, 17):
        check(dev, T, 192, 128, 5, 2, BF16, bits, seed=T)


def test_more_than_sixteen_tokens_and_fp32_over_4_bits(dev):
    """What the two launches do not take runs on the layer's other kernels: the interims are rounded to the type there."""
    for T, dtype, d in ((17, BF16, 128), (40, F16, 192), (5, torch.float32, 96)):
        x, wg, w, (w1, w3, w2) = make(T, d, 128, 4, 2, dtype, 4)
        want, weights, idx, terms, back = oracle.layer(x, wg, w1, w3, w2, 2)
        out, _, ei = run(dev, x, wg, w, 2, bits=4)
        assert torch.equal(ei.cpu().long(), idx)
        u = torch.finfo(dtype).eps / 2
        # gate, up and h are rounded once each: three half steps of |silu'| <= 1.1 gate up
        assert float(((out.double().cpu() - want).abs() - (u * want.abs() + 3.3 * u * (terms + back) + 300 * 2.0 ** -24 * (terms + back))).max()) <= 0


@pytest.mark.parametrize("bits", [16, 4])
def test_ties_go_to_the_lower_expert(dev, bits):
    x, wg, w, _ = make(5, 128, 64, 8, 3, BF16, bits)
    wg[5] = wg[2]
    wg[7] = wg[2]
    wg[2] *= 1
    x[0] = 0                                              # every logit 0
    _, ew, ei = run(dev, x, wg, w, 3, bits=bits)
    _, _, idx = oracle.router(x, wg, 3)
    assert torch.equal(ei.cpu().long(), idx)
    assert ei[0].tolist() == [0, 1, 2] and torch.allclose(ew[0].cpu(), torch.full((3,), 1 / 3))


@pytest.mark.parametrize("bits", [16, 4])
def test_what_is_not_finite_stays_with_its_token(dev, bits):
    T, d, f, E, k = 6, 128, 192, 4, 2
    x, wg, w, _ = make(T, d, f, E, k, BF16, bits)
    clean = run(dev, x, wg, w, k, bits=bits)
    x2 = x.clone()
    x2[2, 5] = float("nan")
    x2[4, 9] = float("inf")
    out, ew, ei = run(dev, x2, wg, w, k, bits=bits)
    assert int(ei.min()) >= 0 and int(ei.max()) < E
    keep = [0, 1, 3, 5]
    for a, b in zip((out, ew, ei), clean):
        assert torch.equal(a[keep], b[keep])
    assert torch.isnan(out[2]).all() and not torch.isfinite(out[4]).any()
    # ... and an expert's weights with those that chose it
    chosen = (clean[2] == 1).any(-1).cpu()
    if bits == 16:
        w[1][1, 3, 7], w[0][1, 8, 2] = float("inf"), float("nan")
    else:
        w[1][1][1, 7, 0], w[0][1][1, 8, 0] = 255, 255
    out, ew, ei = run(dev, x, wg, w, k, bits=bits)
    assert torch.equal(ew, clean[1]) and torch.equal(ei, clean[2])
    assert bool(chosen.any()) and not bool(chosen.all())
    assert torch.equal(out[~chosen], clean[0][~chosen])
    assert not torch.isfinite(out[chosen]).all()


@pytest.mark.parametrize("bits", [16, 4])
def test_repeats_itself_and_in_a_graph(dev, bits):
    T, d, f, E, k = 9, 256, 448, 8, 2
    x, wg, w, _ = make(T, d, f, E, k, BF16, bits)
    xs = [(x + i).to(dev) for i in range(4)]
    wgd = wg.to(dev)
    wd = [t.to(dev) for t in w] if bits == 16 else moe.Fp4ExpertWeights(*(t.to(dev) for q in w for t in q))
    call = (lambda v: moe.moe_layer_decode(v, wgd, *wd, k)) if bits == 16 else (lambda v: moe.moe_layer_forward_fp4(v, wgd, wd, k))
    with torch.no_grad():
        eager = [call(v) for v in xs]
        for v, e in zip(xs, eager):
            for _ in range(5):
                assert all(torch.equal(a, b) for a, b in zip(call(v), e))
        buf = xs[0].clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            call(buf)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call(buf)
        for n in range(8):
            buf.copy_(xs[n % 4])
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, eager[n % 4])), n
            call(xs[(n + 1) % 4])


@pytest.mark.parametrize("bits", [16, 4])
def test_two_calls_at_once(dev, bits):
    T, d, f, E, k = 4, 512, 1024, 8, 2
    x, wg, w, _ = make(T, d, f, E, k, BF16, bits)
    xd = [(x * (i + 1)).to(dev) for i in range(2)]
    wgd = wg.to(dev)
    wd = [t.to(dev) for t in w] if bits == 16 else moe.Fp4ExpertWeights(*(t.to(dev) for q in w for t in q))
    call = (lambda v: moe.moe_layer_decode(v, wgd, *wd, k)) if bits == 16 else (lambda v: moe.moe_layer_forward_fp4(v, wgd, wd, k))
    with torch.no_grad():
        want = [call(v) for v in xd]
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = [[], []]
        for _ in range(20):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i].append(call(xd[i]))
        torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for r in got[i] for a, b in zip(r, want[i]))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_strides_and_unaligned_inputs(dev, dtype):
    T, d, f, E, k = 5, 128, 192, 4, 2
    x, wg, w, _ = make(T, d, f, E, k, dtype, 16)
    want = run(dev, x, wg, w, k)
    with torch.no_grad():
        odd = lambda t: torch.cat((t[..., :3], t), -1)[..., 3:]
        turned = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
        for move in (odd, turned):
            got = moe.moe_layer_decode(move(x.to(dev)), move(wg.to(dev)), *(move(t.to(dev)) for t in w), k)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_agrees_with_the_layer(dev):
    """moe_layer_forward rounds its interims to the type; both lie within a few half steps of each other."""
    x, wg, w, _ = make(8, 256, 512, 8, 2, BF16, 16)
    out, ew, ei = run(dev, x, wg, w, 2)
    with torch.no_grad():
        o2, w2, i2 = moe.moe_layer_forward(x.to(dev), wg.to(dev), *(t.to(dev) for t in w), 2)
    assert torch.equal(ei, i2) and torch.allclose(ew, w2, rtol=1e-5)
    assert float((out.float() - o2.float()).norm() / o2.float().norm()) < 4 * 2.0 ** -8


def test_empty(dev):
    x, wg, w, _ = make(1, 64, 64, 2, 1, BF16, 16)
    with torch.no_grad():
        out, ew, ei = moe.moe_layer_decode(x[:0].to(dev), wg.to(dev), *(t.to(dev) for t in w), 1)
    assert out.shape == (0, 64) and ew.shape == (0, 1) and ei.shape == (0, 1)


def make_codes(T, d, f, E, seed=0):
    """Any codes and scales: what a quantisation gives is a part of them."""
    g = torch.Generator().manual_seed(seed * 31 + T + d + f + E)
    x = torch.randn(T, d, generator=g).to(BF16)
    wg = (torch.randn(E, d, generator=g) * 0.05).to(BF16)
    q = [(torch.randint(0, 256, (E, n, m // 2), generator=g, dtype=torch.uint8), torch.randint(117, 123, (E, n, m // 32), generator=g, dtype=torch.uint8)) for n, m in ((f, d), (d, f), (f, d))]
    return x, wg, q


KEPT = [  # more blocks of 16 ffn columns than the card has compute units, hidden sizes up to 4096 and above
    (3, 512, 1024, 8, 2), (16, 1024, 1024, 8, 2), (5, 1536, 2048, 4, 3), (2, 4096, 1536, 4, 2), (16, 2048, 512, 32, 4), (6, 576, 1216, 6, 3), (9, 128, 2112, 4, 2), (8, 64, 4160, 2, 1),
    (2, 4160, 1088, 4, 2), (1, 8192, 2112, 2, 2), (12, 256, 960, 20, 8),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,d,f,E,k", KEPT)
def test_layer_of_many_blocks(dev, T, d, f, E, k, dtype):
    check(dev, T, d, f, E, k, dtype, 16)


@pytest.mark.parametrize("T,d,f,E,k", KEPT)
def test_layer_of_many_blocks_in_4_bits(dev, T, d, f, E, k):
    x, wg, q = make_codes(T, d, f, E)
    w1, w2, w3 = (oracle.weights(*t, n) for t, n in zip(q, (d, f, d)))
    want, weights, idx, terms, back = oracle.layer(x, wg, w1, w3, w2, k)
    out, ew, ei = run(dev, x, wg, q, k, bits=4)
    assert torch.equal(ei.cpu().long(), idx)
    lt = 2 * ((d + 8) * (x.double().abs() @ wg.double().abs().t()).amax() + 16) * 2.0 ** -24
    assert float(((ew.double().cpu() - weights) / weights).abs().max()) <= lt
    over = (out.double().cpu() - want).abs() - slack_of(want, terms, back, 0.0, d, f, BF16) - lt * terms
    assert float(over.max()) <= 0


@pytest.mark.parametrize("bits", [16, 4])
def test_many_blocks_repeat_and_keep_what_is_not_finite(dev, bits):
    """The same bits from call to call, and from a token alone to the same token beside others that hold NaN."""
    T, d, f, E, k = 10, 512, 1536, 6, 2
    x, wg, q = make_codes(T, d, f, E)
    w = q if bits == 4 else [(0.05 * torch.randn(E, f, d, generator=torch.Generator().manual_seed(i))).to(BF16) for i in range(3)]
    want = run(dev, x, wg, w, k, bits=bits)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(run(dev, x, wg, w, k, bits=bits), want))
    bad = x.clone()
    bad[3], bad[7, 100] = float("nan"), float("-inf")
    out, ew, ei = run(dev, bad, wg, w, k, bits=bits)
    keep = [0, 1, 2, 4, 5, 6, 8, 9]
    assert torch.equal(out[keep], want[0][keep]) and torch.equal(ei[keep], want[2][keep]) and int(ei.min()) >= 0 and int(ei.max()) < E


def test_codes_and_scales_at_odd_addresses(dev):
    T, d, f, E, k = 4, 512, 1024, 8, 2
    x, wg, q = make_codes(T, d, f, E)
    want = run(dev, x, wg, q, k, bits=4)

    def odd(t):
        buf = torch.empty(t.numel() + 16, dtype=t.dtype, device=dev)
        at = 3 if buf.data_ptr() % 16 == 0 else 0
        return buf[at:at + t.numel()].view(t.shape).copy_(t)
    with torch.no_grad():
        for pick in (lambda i: True, lambda i: i % 2 == 0, lambda i: i % 2 == 1):
            w = moe.Fp4ExpertWeights(*(odd(t) if pick(i) else t.to(dev) for i, t in enumerate(t for p in q for t in p)))
            got = moe.moe_layer_forward_fp4(x.to(dev), wg.to(dev), w, k)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        # one row of a pitch that 16-byte loads do not take, and every token the same row
        one = torch.empty(1, d + 3, dtype=BF16, device=dev)[:, :d].copy_(x[:1])
        assert torch.equal(moe.moe_layer_forward_fp4(one, wg.to(dev), moe.Fp4ExpertWeights(*(t.to(dev) for p in q for t in p)), k)[0], run(dev, x[:1], wg, q, k, bits=4)[0])
        same = moe.moe_layer_forward_fp4(x[:1].to(dev).expand(5, d), wg.to(dev), moe.Fp4ExpertWeights(*(t.to(dev) for p in q for t in p)), k)[0]
        assert torch.equal(same, run(dev, x[:1].repeat(5, 1), wg, q, k, bits=4)[0])


def test_graphs_that_share_a_memory_pool(dev):
    """Two captured layers whose workspaces may be the same memory, replayed in turn between eager calls."""
    T, d, f, E, k = 5, 512, 1024, 8, 2
    x, wg, q = make_codes(T, d, f, E)
    xd, wgd, w4 = x.to(dev), wg.to(dev), moe.Fp4ExpertWeights(*(t.to(dev) for p in q for t in p))
    w16 = [(0.05 * torch.randn(E, f, d, generator=torch.Generator().manual_seed(i))).to(BF16).to(dev) for i in range(3)]
    calls = [lambda: moe.moe_layer_forward_fp4(xd, wgd, w4, k)[0], lambda: moe.moe_layer_decode(xd, wgd, *w16, k)[0]]
    with torch.no_grad():
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
            xd.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(trial)).to(BF16))
            graphs[i].replay()
            torch.cuda.synchronize()
            got = outs[i].clone()
            assert torch.equal(got, calls[i]()), (trial, i)


# ---------------------------------------------------------------------------------------------------------------
# the router of the few-token layer beside the framework's own
# ---------------------------------------------------------------------------------------------------------------
def route_both(dev, x, wg, k, f, normalize=True, bits=4):
    """(weights, indices) of the few-token layer, and of the router that every other path takes."""
    E, d = wg.shape
    if bits == 16:
        w = [torch.zeros(E, f, d, dtype=x.dtype) for _ in range(3)]
    else:
        w = [(torch.zeros(E, n, m // 2, dtype=torch.uint8), torch.full((E, n, m // 32), 120, dtype=torch.uint8)) for n, m in ((f, d), (d, f), (f, d))]
    few = run(dev, x, wg, w, k, normalize, bits)
    return few[1:], moe.megablocks_utils.router.router_forward(x.to(dev), wg.to(dev), k, normalize)[2:]


def with_logits(logits, d, dtype, rest=None):
    """x (T, d) and wg (E, d) whose logits are the given ones (numbers of the type), plus `rest` where given: sums of one or two exact products."""
    T, E = logits.shape
    x, wg = torch.zeros(T, d, dtype=dtype), torch.zeros(E, d, dtype=dtype)
    at = torch.arange(T)
    x[at, at] = 1
    wg[:, :T] = logits.t().to(dtype)
    assert torch.equal(wg[:, :T].double(), logits.t().double())
    if rest is not None:
        x[at, T + at] = 1
        wg[:, T:2 * T] = rest.t().to(dtype)
        assert torch.equal(wg[:, T:2 * T].double(), rest.t().double())
    return x, wg


@pytest.mark.parametrize("E,k,d,f", [(8, 4, 128, 64), (8, 8, 1024, 1088), (24, 6, 512, 1088), (64, 8, 192, 64), (200, 16, 4160, 64)])
@pytest.mark.parametrize("normalize", [True, False])
def test_scores_that_underflow_are_ties(dev, E, k, d, f, normalize):
    """Experts are ranked by their fp32 scores: exp(-110) and less is 0 in fp32 (the least subnormal number is e^-103.3), so all but the first ones tie, and ties go to the lower
    expert."""
    g = torch.Generator().manual_seed(E)
    T = 7
    logits = -110.0 - torch.randint(0, 16, (T, E), generator=g).double()
    best = [torch.randperm(E, generator=g)[:n % 3 + 1].tolist() for n in range(T)]
    for t, b in enumerate(best):
        for j, e in enumerate(b):
            logits[t, e] = 8.0 - j
    x, wg = with_logits(logits, d, BF16)
    (ew, ei), (rw, ri) = route_both(dev, x, wg, k, f, normalize)
    for t, b in enumerate(best):
        assert ei[t].tolist() == (b + [e for e in range(E) if e not in b])[:k], t
        assert not ew[t, len(b):].any()
    assert torch.equal(ei, ri) and torch.equal(ew, rw)


@pytest.mark.parametrize("E,k", [(8, 3), (16, 16), (64, 8)])
def test_logits_that_round_to_one_score(dev, E, k):
    """Neighbouring fp32 numbers below -1: their exponentials are spaced more widely than they are apart."""
    g = torch.Generator().manual_seed(E)
    T = 9
    rest = torch.stack([torch.randperm(E, generator=g) for _ in range(T)]).double() * 2.0 ** -24
    base = torch.full((T, E), -1.0).double()
    base[torch.arange(T), torch.randint(0, E, (T,), generator=g)] = torch.arange(T).double() / 4
    x, wg = with_logits(base, 128, BF16, rest)
    (ew, ei), (rw, ri) = route_both(dev, x, wg, k, 64)
    assert torch.equal(ei, ri) and torch.equal(ew, rw)


@pytest.mark.parametrize("E,k", [(4, 2), (12, 5), (64, 8)])
def test_tokens_without_finite_scores_take_experts_in_order(dev, E, k):
    """A NaN among the logits, or an infinite one: every score of the token is NaN, which loses to no other, and its experts are the first ones; as in every other path."""
    T, d = 6, 128
    g = torch.Generator().manual_seed(E)
    x, wg = with_logits(torch.randint(-8, 9, (T, E), generator=g).double(), d, BF16)
    x[1, 100], wg[E - 1, 100] = 2.0 ** 100, 2.0 ** 100      # one logit overflows to infinity
    x[2, 101], wg[2, 101] = -2.0 ** 100, 2.0 ** 100         # one is minus infinity: a score of 0
    x[3, 102] = float("nan")
    (ew, ei), (rw, ri) = route_both(dev, x, wg, k, 64)
    for t in (1, 3):
        assert ei[t].tolist() == list(range(k)) and torch.isnan(ew[t]).all()
    assert torch.isfinite(ew[2]).all() and 2 not in ei[2].tolist()
    assert torch.equal(ei, ri) and torch.equal(torch.nan_to_num(ew, 7.0), torch.nan_to_num(rw, 7.0))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("d,f,at", [(1024, 384, (0, 1, 2, 3)), (1024, 64, (0, 1, 2, 3)), (4096, 384, (12, 13, 14, 15)), (4224, 128, (0, 8, 16, 24))])
def test_large_terms_that_cancel_do_not_hide_the_others(dev, d, f, at, bits, dtype):
    """Logits are 2^16 r 2^-25 + 2^16 - 2^16 over 16 experts: 256 terms r 2^-17 between two that cancel, in chunks of 128 inputs of one wave's share.  A sum of 32 terms is exact in fp32 (and lost in a
    fp32 sum that already holds 2^16: at most 15 * 2^-12 < half of its last place, 2^-8)."""
    E, k, T = 16, 8, 3
    g = torch.Generator().manual_seed(d + f)
    ranks = torch.randperm(E, generator=g)
    x, wg = torch.zeros(T, d, dtype=dtype), torch.zeros(E, d, dtype=dtype)
    for t in range(T):
        x[t, at[0] * 128 + 5], x[t, at[3] * 128 + 77] = 256, -256
        x[t, at[1] * 128:at[1] * 128 + 128] = x[t, at[2] * 128:at[2] * 128 + 128] = 1
    wg[:, at[0] * 128 + 5] = wg[:, at[3] * 128 + 77] = 256
    for c in at[1:3]:
        wg[:, c * 128:c * 128 + 128] = (ranks.double() * 2.0 ** -17).to(dtype)[:, None]
    _, weights, idx = oracle.router(x, wg, k)
    assert torch.equal(idx[0], ranks.argsort(descending=True)[:k])
    (ew, ei), (rw, ri) = route_both(dev, x, wg, k, f, bits=bits)
    assert torch.equal(ri.cpu().long(), idx)
    assert torch.equal(ei.cpu().long(), idx)
    # logits are exact; an exponential within 2^-23, a sum and two quotients on top
    assert float(((ew.double().cpu() - weights) / weights).abs().max()) <= 24 * 2.0 ** -24


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,d,f,E,k", KEPT + [(8, 2048, 1024, 64, 8), (1, 512, 4160, 2, 1), (11, 3584, 1536, 4, 2)])
def test_layer_of_many_blocks_in_4_bits_of_either_type(dev, T, d, f, E, k, dtype):
    """Scales 117 to 122 are exact in both types."""
    x, wg, q = make_codes(T, d, f, E)
    x, wg = x.to(dtype), wg.to(dtype)
    w1, w2, w3 = (oracle.weights(*t, n) for t, n in zip(q, (d, f, d)))
    want, weights, idx, terms, back = oracle.layer(x, wg, w1, w3, w2, k)
    out, ew, ei = run(dev, x, wg, q, k, bits=4)
    assert out.dtype == dtype and torch.equal(ei.cpu().long(), idx)
    lt = 2 * ((d + 8) * (x.double().abs() @ wg.double().abs().t()).amax() + 16) * 2.0 ** -24
    assert float(((ew.double().cpu() - weights) / weights).abs().max()) <= lt
    w2_sum = sum((w2[idx[:, j]].abs().sum(-1) * weights[:, j, None]) for j in range(k))
    over = (out.double().cpu() - want).abs() - slack_of(want, terms, back, w2_sum, d, f, dtype) - lt * terms
    assert float(over.max()) <= 0
