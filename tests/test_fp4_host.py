"""The layers over 4-bit weights, for a few tokens and the SwiGLU that keeps 8-bit inputs on the host: what their entry points refuse before anything is enqueued (tensors
are fakes that only claim to lie on a GPU), what the C entries refuse, and the 64-bit oracle against closed forms."""
import warnings

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import moe_distributed_training_amd as moe
from oracle import fp4_oracle as oracle

T, K, N, E, k = 24, 64, 128, 4, 2
BF16, F16, F32, U8, I8, I32 = torch.bfloat16, torch.float16, torch.float32, torch.uint8, torch.int8, torch.int32
_MODE = FakeTensorMode(allow_non_fake_inputs=True)
on_host = pytest.mark.skipif(torch.cuda.is_available(), reason="a fake's pointer must not reach a kernel")
ELSEWHERE = [("GPU only", "cpu"), ("same device", "cuda:1")]


def _fake(*shape, dtype=BF16, device="cuda:0", grad=False):
    with _MODE:
        return torch.empty(shape, dtype=dtype, device=device, requires_grad=grad)


def _refused(match, fn, *args, **kw):
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")   # (a fake's data pointer)
        with pytest.raises((RuntimeError, AssertionError, TypeError), match=match):
            fn(*args, **kw)


def _linear(**changed):
    args = dict(inputs=_fake(T, K), expert_codes=_fake(E, N, K // 2, dtype=U8), weight_scales=_fake(E, N, K // 32, dtype=U8), k=k, sorted_expert_idxs=_fake(T * k, dtype=I32),
                sorted_scattered_idxs=_fake(T * k, dtype=I32), padded_block_idxs=None, expert_offsets=_fake(E, dtype=I32))
    return moe.parallel_linear_fp4, {**args, **changed}


def _weights(d=K, f=N, **changed):
    w = dict(w1=_fake(E, f, d // 2, dtype=U8), w1_scale=_fake(E, f, d // 32, dtype=U8), w2=_fake(E, d, f // 2, dtype=U8), w2_scale=_fake(E, d, f // 32, dtype=U8),
             w3=_fake(E, f, d // 2, dtype=U8), w3_scale=_fake(E, f, d // 32, dtype=U8))
    return moe.Fp4ExpertWeights(**{**w, **changed})


def _mlp(weights=None, **changed):
    args = dict(x=_fake(T, K), weights=weights or _weights(), k=k, sorted_scattered_idxs=_fake(T * k, dtype=I32), expert_offsets=_fake(E, dtype=I32))
    return moe.fused_expert_mlp_fp4, {**args, **changed}


def _decode(**changed):
    args = dict(x=_fake(4, K), wg=_fake(E, K), w1=_fake(E, N, K), w2=_fake(E, N, K), w3=_fake(E, N, K), top_k=k)
    return moe.moe_layer_decode, {**args, **changed}


@on_host
@pytest.mark.parametrize("match,device", ELSEWHERE)
@pytest.mark.parametrize("name,shape,dtype", [("expert_codes", (E, N, K // 2), U8), ("weight_scales", (E, N, K // 32), U8), ("sorted_expert_idxs", (T * k,), I32),
                                              ("sorted_scattered_idxs", (T * k,), I32), ("expert_offsets", (E,), I32), ("gates", (T, k), F32)])
def test_projection_tensors_elsewhere(match, device, name, shape, dtype):
    fn, args = _linear(**{name: _fake(*shape, dtype=dtype, device=device)})
    _refused(match, fn, **args)


@on_host
@pytest.mark.parametrize("match,changed", [
    ("has to be", dict(inputs=_fake(T, K, 1))), ("nothing to multiply", dict(inputs=_fake(T, 0))), ("are not 4-bit weights of 96 inputs", dict(inputs=_fake(T, 96))),
    ("uint8, two to a byte", dict(expert_codes=_fake(E, N, K // 2, dtype=I8))), ("uint8 exponents", dict(weight_scales=_fake(E, N, K // 32, dtype=F32))),
    ("experts, outputs", dict(expert_codes=_fake(N, K // 2, dtype=U8))), ("experts, outputs", dict(weight_scales=_fake(E, N, dtype=U8))),
    ("are not 4-bit weights", dict(weight_scales=_fake(E, N - 1, K // 32, dtype=U8))), ("are not 4-bit weights", dict(expert_codes=_fake(E, N, K, dtype=U8))),
    ("are not 4-bit weights", dict(weight_scales=_fake(E + 1, N, K // 32, dtype=U8))), ("hold nothing", dict(expert_codes=_fake(0, N, K // 2, dtype=U8), weight_scales=_fake(0, N, K // 32, dtype=U8))),
    ("unsupported dtype", dict(inputs=_fake(T, K, dtype=torch.float64))), ("unsupported dtype", dict(inputs=_fake(T, K, dtype=I8))), ("assignments", dict(k=3)), ("assignments", dict(k=0)),
    ("length", dict(sorted_expert_idxs=_fake(T, dtype=I32))), ("k is 1", dict(grouped_in=True)), ("cover", dict(expert_offsets=_fake(E - 1, dtype=I32))),
    ("int32 or int64", dict(expert_offsets=_fake(E, dtype=F32))), ("int32 or int64", dict(sorted_scattered_idxs=_fake(T * k, dtype=torch.int16))),
    ("gates of", dict(gates=_fake(T * k, dtype=F32))), ("gates of", dict(gates=_fake(T, k + 1, dtype=F32))), ("grouped output", dict(gates=_fake(T, k, dtype=F32), grouped_out=True)),
    ("unsupported dtype", dict(gates=_fake(T, k, dtype=torch.float64)))])
def test_projection_arguments(match, changed):
    fn, args = _linear(**changed)
    _refused(match, fn, **args)


@on_host
@pytest.mark.parametrize("match,device", ELSEWHERE)
@pytest.mark.parametrize("name", moe.Fp4ExpertWeights._fields)
def test_mlp_weights_elsewhere(match, device, name):
    t = getattr(_weights(), name)
    w = _weights(**{name: _fake(*t.shape, dtype=t.dtype, device=device)})
    fn, args = _mlp(w)
    _refused(match, fn, **args)
    _refused(match, moe.moe_layer_forward_fp4, _fake(4, K), _fake(E, K), w)


@on_host
@pytest.mark.parametrize("match,weights,changed", [
    ("do not fit", dict(w2=_fake(E, K + 64, N // 2, dtype=U8), w2_scale=_fake(E, K + 64, N // 32, dtype=U8)), {}),
    ("do not fit", dict(w3=_fake(E + 1, N, K // 2, dtype=U8), w3_scale=_fake(E + 1, N, K // 32, dtype=U8)), {}), ("two to a byte", dict(w1=_fake(E, N, K // 2)), {}),
    ("are not 4-bit weights", dict(w2=_fake(E, N, K // 2, dtype=U8), w2_scale=_fake(E, N, K // 32, dtype=U8)), {}), ("exponents", dict(w2_scale=_fake(E, K, N // 32, dtype=F32)), {}),
    ("unsupported dtype", {}, dict(x=_fake(T, K, dtype=torch.float64))), ("are not 4-bit weights", {}, dict(x=_fake(T, K + 64))), ("do not fit", {}, dict(k=1)), ("do not fit", {}, dict(k=0)),
    ("hidden size", {}, dict(x=_fake(T, K, 1))), ("cover", {}, dict(expert_offsets=_fake(E - 1, dtype=I32))), ("int32 or int64", {}, dict(sorted_scattered_idxs=_fake(T * k, dtype=F32))),
    ("gates of", {}, dict(gates=_fake(k, T, 1, dtype=F32)))])
def test_mlp_arguments(match, weights, changed):
    fn, args = _mlp(_weights(**weights), **changed)
    _refused(match, fn, **args)


@on_host
def test_layer_arguments():
    _refused("router weight", moe.moe_layer_forward_fp4, _fake(T, K), _fake(E + 1, K), _weights())
    _refused("share a dtype", moe.moe_layer_forward_fp4, _fake(T, K), _fake(E, K, dtype=F32), _weights())
    _refused("top_k", moe.moe_layer_forward_fp4, _fake(T, K), _fake(E, K), _weights(), E + 1)
    _refused("top_k", moe.moe_layer_forward_fp4, _fake(T, K), _fake(E, K), _weights(), 0)
    _refused("hidden size", moe.moe_layer_forward_fp4, _fake(T, K, 1), _fake(E, K), _weights())
    _refused("experts, inputs, outputs", moe.quantize_expert_weights_fp4, _fake(T, K))
    _refused("unsupported dtype", moe.quantize_expert_weights_fp4, _fake(E, K, N, dtype=I8))
    _refused("GPU only", moe.quantize_expert_weights_fp4, torch.zeros(2, 3, 4))


@on_host
@pytest.mark.parametrize("match,device", ELSEWHERE)
@pytest.mark.parametrize("name", ["wg", "w1", "w2", "w3"])
def test_decode_tensors_elsewhere(match, device, name):
    fn, args = _decode()
    args[name] = _fake(*args[name].shape, device=device)
    _refused(match, fn, **args)


@on_host
@pytest.mark.parametrize("match,changed", [
    ("up to 16 tokens", dict(x=_fake(17, K))), ("use moe_layer_forward", dict(top_k=17, wg=_fake(32, K), w1=_fake(32, N, K), w2=_fake(32, N, K), w3=_fake(32, N, K))),
    ("256 experts", dict(wg=_fake(257, K), w1=_fake(257, N, K), w2=_fake(257, N, K), w3=_fake(257, N, K))),
    ("multiples of 64", dict(x=_fake(4, 96), wg=_fake(E, 96), w1=_fake(E, N, 96), w2=_fake(E, N, 96), w3=_fake(E, N, 96))),
    ("multiples of 64", dict(w1=_fake(E, 100, K), w2=_fake(E, 100, K), w3=_fake(E, 100, K))), ("below 2 GiB", dict(w1=_fake(E, 1 << 21, K), w2=_fake(E, 1 << 21, K), w3=_fake(E, 1 << 21, K))),
    ("multiples of 64", dict(w1=_fake(E, 0, K), w2=_fake(E, 0, K), w3=_fake(E, 0, K))),
    ("bf16 or fp16", dict(x=_fake(4, K, dtype=F32), wg=_fake(E, K, dtype=F32), w1=_fake(E, N, K, dtype=F32), w2=_fake(E, N, K, dtype=F32), w3=_fake(E, N, K, dtype=F32))),
    ("share a dtype", dict(wg=_fake(E, K, dtype=F16))), ("share a dtype", dict(w2=_fake(E, N, K, dtype=F16))), ("router weight", dict(wg=_fake(E, K + 64))), ("router weight", dict(wg=_fake(K))),
    ("expert weight", dict(w2=_fake(E, K, N))), ("expert weight", dict(w1=_fake(E * N, K))), ("expert weights are", dict(w3=_fake(E * N, K))), ("top_k", dict(top_k=0)), ("top_k", dict(top_k=E + 1)),
    ("tokens, hidden size", dict(x=_fake(4, 1, K))), ("no gradients", dict(x=_fake(4, K, grad=True))), ("no gradients", dict(w2=_fake(E, N, K, grad=True)))])
def test_decode_arguments(match, changed):
    fn, args = _decode(**changed)
    _refused(match, fn, **args)


@on_host
def test_swiglu_arguments():
    g = _fake(T, K)
    _refused("differ in shape", moe.swiglu_8bit, g, _fake(T, K + 1))
    _refused("differ in shape", moe.swiglu_8bit, _fake(), _fake())
    _refused("share a dtype", moe.swiglu_8bit, g, _fake(T, K, dtype=F16))
    _refused("unsupported dtype", moe.swiglu_8bit, _fake(T, K, dtype=torch.float64), _fake(T, K, dtype=torch.float64))
    _refused("same device", moe.swiglu_8bit, g, _fake(T, K, device="cuda:1"))
    _refused("GPU only", moe.swiglu_8bit, torch.zeros(2, 3), torch.zeros(2, 3))


def test_c_entries_refuse_on_the_host():
    """Status codes before anything is enqueued (16 and 256: non-null stand-ins that are never dereferenced)."""
    from moe_distributed_training_amd._lib import lib
    BAD, UNSUP, SPACE = -1, -2, -3

    def quant(w=16, dt=0, E=2, K=64, N=128, c=16, sce=4096, scn=32, s=16):
        return lib.moe_fp4_quantize_weights(w, K * N, N, 1, dt, E, K, N, c, sce, scn, s, 256, 2, None)
    assert all(v == BAD for v in (quant(w=None), quant(c=None), quant(s=None), quant(dt=3), quant(dt=-1), quant(E=0), quant(K=0), quant(N=0), quant(c=24), quant(scn=16), quant(scn=40), quant(sce=8)))

    def fwd(x=16, ldx=64, rows=8, dt=0, c=16, sce=4096, scn=32, s=16, y=16, ldy=128, ydt=0, pos=16, off=16, E=2, R=16, K=64, N=128, fan=2, xg=0, yg=0, ws=256, n=1 << 40):
        return lib.moe_linear_fp4_fwd(x, ldx, rows, dt, c, sce, scn, s, 256, 2, y, ldy, ydt, pos, 0, off, 0, E, R, K, N, fan, xg, yg, ws, n, None)
    assert all(v == BAD for v in (fwd(x=None), fwd(c=None), fwd(c=24), fwd(scn=24), fwd(sce=8), fwd(s=None), fwd(y=None), fwd(pos=None), fwd(off=None), fwd(dt=3), fwd(ydt=-1), fwd(ldx=-1),
                                  fwd(ldy=127), fwd(E=0), fwd(R=-1), fwd(K=0), fwd(N=-1), fwd(fan=0), fwd(rows=-1), fwd(rows=0), fwd(xg=1, rows=15), fwd(ws=24)))
    assert fwd(R=0, x=None) == 0 and fwd(N=0, y=None) == 0
    # scales of two groups and no multiple of four are copied into rows of four: 2 experts x 128 columns x 4; nothing where both lie well
    assert lib.moe_linear_fp4_workspace_bytes(16, 64, 8, 0, 0, 16, 256, 2, 16, 2, 64, 128) == 1024 and lib.moe_linear_fp4_workspace_bytes(16, 128, 8, 0, 0, 16, 512, 4, 16, 2, 128, 128) == 0
    assert lib.moe_linear_fp4_workspace_bytes(18, 65, 8, 0, 2, 17, 255, 2, 16, 2, 65, 128) == 0                            # fp32 takes everything as it lies
    assert fwd(n=1023) == SPACE and fwd(ws=None) == SPACE
    assert lib.moe_linear_fp4_workspace_bytes(16, 65, 8, 0, 0, 16, 512, 4, 16, 2, 128, 128) == 16 * 128 * 2 and lib.moe_linear_fp4_workspace_bytes(18, 128, 8, 0, 0, 16, 512, 4, 16, 2, 128, 128) == 16 * 128 * 2
    assert lib.moe_linear_fp4_workspace_bytes(16, 64, 8, 0, 5, 16, 256, 2, 16, 2, 64, 128) == 0 and lib.moe_linear_fp4_workspace_bytes(16, 64, 8, 0, 0, 16, 256, 2, 0, 2, 64, 128) == 0
    assert fwd(dt=2, ydt=0) == UNSUP and fwd(K=1 << 22, ldx=1 << 22, scn=1 << 21, sce=1 << 28) == UNSUP and fwd(N=1 << 27, ldy=1 << 27) == UNSUP

    def bwd(dy=16, ldd=128, rows=8, dt=0, dg=0, fan=2, gates=None, gdt=0, c=16, scn=32, s=16, dx=16, ldx=64, dxt=0, xg=0, pos=16, off=16, E=2, R=16, K=64, N=128, ws=256, n=1 << 40):
        return lib.moe_linear_fp4_bwd(dy, ldd, rows, dt, dg, fan, gates, gdt, c, 4096, scn, s, 256, 2, dx, ldx, dxt, xg, pos, 0, off, 0, E, R, K, N, ws, n, None)
    assert all(v == BAD for v in (bwd(dy=None), bwd(ldd=-1), bwd(rows=0), bwd(dt=3), bwd(dxt=3), bwd(gates=16, gdt=3), bwd(gates=16, dg=1, rows=16), bwd(c=24), bwd(scn=8), bwd(s=None),
                                  bwd(dx=None), bwd(ldx=63), bwd(pos=None), bwd(off=None), bwd(E=0), bwd(K=0), bwd(N=0), bwd(fan=0), bwd(dg=1, rows=15), bwd(ws=8)))
    assert bwd(R=0, dy=None) == 0 and bwd(n=1023) == SPACE and bwd(ws=None) == SPACE and bwd(dt=2, dxt=0) == UNSUP
    assert lib.moe_linear_fp4_bwd_workspace_bytes(16, 128, 8, 0, 0, 16, 512, 4, 16, 2, 128, 128) == 0
    assert lib.moe_linear_fp4_bwd_workspace_bytes(16, 130, 8, 0, 0, 16, 512, 4, 16, 2, 128, 130) == 16 * 136 * 2

    kept = lib.moe_swiglu8_kept_bytes(3, 65)
    assert kept == 2 * (512 + 256) and lib.moe_swiglu8_kept_bytes(0, 65) == 0 and lib.moe_swiglu8_kept_bytes(3, -1) == 0   # three rows of two blocks of 64 codes, a scale each; pieces of 256

    def sf(g=16, ldg=65, u=16, ldu=65, h=16, ldh=65, kp=256, n=kept, rows=3, cols=65, dt=0):
        return lib.moe_swiglu8_fwd(g, ldg, u, ldu, h, ldh, kp, n, rows, cols, dt, None)

    def sb(kp=256, n=kept, dh=16, ld=65, a=16, lda=65, b=16, ldb=65, rows=3, cols=65, dt=0):
        return lib.moe_swiglu8_bwd(kp, n, dh, ld, a, lda, b, ldb, rows, cols, dt, None)
    assert all(v == BAD for v in (sf(g=None), sf(u=None), sf(h=None), sf(ldg=-1), sf(ldu=-1), sf(ldh=64), sf(kp=24), sf(rows=-1), sf(cols=-1), sf(dt=3)))
    assert all(v == BAD for v in (sb(kp=None), sb(dh=None), sb(a=None), sb(b=None), sb(ld=-1), sb(lda=64), sb(ldb=64), sb(kp=24), sb(rows=-1), sb(dt=-1)))
    assert sf(n=kept - 1) == SPACE and sb(n=kept - 1) == SPACE and sf(rows=0, g=None) == 0 and sb(cols=0, kp=None) == 0 and sf(rows=1 << 27, n=1 << 40) == UNSUP and sb(rows=1 << 27, n=1 << 40) == UNSUP

    def dec(x=16, ldx=64, wg=16, ldwg=64, dt=0, w=16, out=16, ldo=64, wt=16, ix=16, T=4, E=4, d=64, f=128, k=2, ws=256, n=1 << 30, four=False, s=16):
        if four:
            return lib.moe_decode_layer_fp4(x, ldx, wg, ldwg, dt, w, s, 16, 16, 16, 16, out, ldo, wt, ix, T, E, d, f, k, 1, ws, n, None)
        return lib.moe_decode_layer(x, ldx, wg, ldwg, dt, w, 16, 16, out, ldo, wt, ix, T, E, d, f, k, 1, ws, n, None)
    for four in (False, True):
        c = lambda **kw: dec(four=four, **kw)
        assert all(v == BAD for v in (c(x=None), c(wg=None), c(w=None), c(out=None), c(wt=None), c(ix=None), c(x=24), c(wg=24), c(w=24), c(out=20), c(ldx=60), c(ldwg=60), c(ldo=62), c(ldo=60),
                                      c(ldx=-64), c(dt=3), c(T=-1), c(E=0), c(d=96), c(f=100), c(d=0), c(k=0), c(k=5), c(ws=24)))
        assert all(v == UNSUP for v in (c(dt=2), c(T=17), c(E=257), c(k=17, E=32), c(d=(1 << 20) + 64), c(ldx=1 << 30), c(ldwg=1 << 29), c(d=1 << 16, f=1 << 15, ldx=1 << 16, ldwg=1 << 16, ldo=1 << 16)))
        need = lib.moe_decode_layer_workspace_bytes(4, 4, 64, 128, 2, 4 if four else 16)
        assert need >= 2 * 4 * 2 * 128 * 2 and c(n=need - 1) == SPACE and c(ws=None) == SPACE and c(T=0, x=None, w=None) == 0
    assert dec(four=True, s=24) == BAD and dec(four=True, s=None) == BAD
    q = lib.moe_decode_layer_workspace_bytes
    assert q(0, 4, 64, 128, 2, 16) == 0 and q(17, 4, 64, 128, 2, 16) == 0 and q(4, 4, 64, 128, 5, 16) == 0 and q(4, 257, 64, 128, 2, 4) == 0


def test_c_entries_refuse_strides_below_zero():
    """Offsets into an expert's codes and scales are unsigned: a negative pitch of 16-bit products would read zeros (stand-ins as above)."""
    from moe_distributed_training_amd._lib import lib
    for dt in (0, 1, 2):
        for sce, scn, sse, ssn in ((-4096, 32, 256, 4), (4096, -32, 256, 4), (4096, 32, -256, 4), (4096, 32, 256, -4)):
            assert lib.moe_linear_fp4_fwd(16, 64, 8, dt, 16, sce, scn, 16, sse, ssn, 16, 128, dt, 16, 0, 16, 0, 2, 16, 64, 128, 2, 0, 0, 256, 1 << 40, None) == -1
            assert lib.moe_linear_fp4_bwd(16, 128, 8, dt, 0, 2, None, 0, 16, sce, scn, 16, sse, ssn, 16, 64, dt, 0, 16, 0, 16, 0, 2, 16, 64, 128, 256, 1 << 40, None) == -1


def test_block_refusals_on_the_host():
    block = moe.ScatterMoEBlock(64, 128, 2, dtype=BF16)
    for match, kw in (("8 or 4 bits", dict(bits=2)), ("goes with experts in 4 bits", dict(keep_8bit=True)), ("goes with experts in 4 bits", dict(bits=8, keep_8bit=True))):
        with pytest.raises(ValueError, match=match):
            block.quantize_experts(**kw)
    for match, kw in (("lora_r = 0", dict(lora_r=4)), ("bf16, fp16 or fp32", dict(dtype=torch.float64)), ("2\\^20", dict(hidden_size=(1 << 20) + 32, num_experts=1, device="meta")),
                      ("2\\^31", dict(hidden_size=1 << 16, ffn_hidden_size=1 << 15, num_experts=1, device="meta"))):
        b = moe.ScatterMoEBlock(**{**dict(hidden_size=64, ffn_hidden_size=128, num_experts=2, dtype=BF16), **kw})
        before = {n: p for n, p in b.named_parameters()}
        with pytest.raises(ValueError, match=match):
            b.quantize_experts(bits=4)
        assert not b.is_quantized and all(dict(b.named_parameters())[n] is p for n, p in before.items())
    with pytest.raises(ValueError, match="without adapters"):
        moe.ScatterMoEBlock(64, 128, 2, lora_r=4, dtype=BF16).decode(torch.zeros(1, 64, dtype=BF16))
    with pytest.raises(RuntimeError, match="GPU only"):
        block.quantize_experts(bits=4)
    assert not block.is_quantized and block.expert_bits == 16 and isinstance(block.w1, torch.nn.Parameter)


def test_a_block_in_4_bits_converts_and_is_not_quantised_twice():
    block = moe.ScatterMoEBlock(64, 128, 2, dtype=BF16)
    for n, rows, cols in (("w1", 128, 64), ("w2", 64, 128), ("w3", 128, 64)):                       # as quantize_experts(bits=4) leaves them
        delattr(block, n)
        block.register_buffer(n, torch.randint(0, 256, (2, rows, cols // 2), dtype=U8))
        block.register_buffer(n + "_scale", torch.randint(110, 130, (2, rows, cols // 32), dtype=U8))
    before = {n: t.clone() for n, t in block.state_dict().items() if n != "router"}
    assert block.is_quantized and block.expert_bits == 4
    block = torch.nn.Sequential(block).half().float().to(BF16)[0]                                    # codes have no type to lose
    assert block.router.dtype == BF16 and all(torch.equal(block.state_dict()[n], t) and block.state_dict()[n].dtype == U8 for n, t in before.items())
    assert block.quantize_experts(bits=4, keep_8bit=True) is block and block.keep_8bit
    with pytest.raises(ValueError, match="4 bits already"):
        block.quantize_experts()


# ---- the oracle itself
def test_oracle_codes():
    """All sixteen codes in one group, units of 2^-3; largest magnitudes 7 units (kept) and just above (the next power); ties to the even code."""
    levels = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    w = torch.zeros(1, 32, 4, dtype=torch.float64)
    w[0, :16, 0] = torch.tensor(levels + [-v for v in levels]) / 8
    w[0, 0, 1], w[0, 0, 2] = 7.0, 7.001
    w[0, :9, 3] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.75, 6.0])
    codes, scales = oracle.quantize(w)
    assert scales[0, :, 0].tolist() == [124, 127, 128, 127]
    nib = lambda n: [int(v) for b in codes[0, n].tolist() for v in (b & 15, b >> 4)]
    assert nib(0)[:16] == [0, 1, 2, 3, 4, 5, 6, 7, 0, 9, 10, 11, 12, 13, 14, 15] and nib(1)[0] == 7 and nib(2)[0] == 6
    assert nib(3)[:9] == [0, 2, 2, 4, 4, 6, 6, 10, 7]
    assert torch.equal(oracle.weights(codes, scales, 32)[0, 0, :16], w[0, :16, 0].abs() * torch.tensor([1.0] * 8 + [-1.0] * 8).double())
    codes, scales = oracle.quantize(torch.tensor([[[float("inf")]], [[float("nan")]], [[0.0]]]))
    assert scales.flatten().tolist() == [255, 255, 0] and int(codes.sum()) == 0 and torch.isnan(oracle.weights(codes, scales, 1)[:2]).all()


def test_oracle_gradients_are_autograds():
    g = torch.Generator().manual_seed(1)
    T_, K_, N_, E_, k_ = 7, 12, 10, 3, 2
    sei, ssi, _, gates = oracle.route(T_, E_, k_, 0)
    w = oracle.weights(*oracle.quantize(torch.randn(E_, K_, N_, generator=g)), K_)
    x, dout = torch.randn(T_, K_, generator=g).double().requires_grad_(True), torch.randn(T_, N_, generator=g).double()
    gw = gates.double().requires_grad_(True)
    expert = torch.empty(T_ * k_, dtype=torch.long)
    expert[ssi] = sei.long()
    rows = torch.stack([w[e] @ x[m // k_] for m, e in enumerate(expert.tolist())])
    y = (rows.view(T_, k_, N_) * gw.unsqueeze(-1)).sum(1)
    dx, dg = torch.autograd.grad(y, (x, gw), dout)
    want = oracle.linear(x.detach(), w, k_, sei, ssi, gw.detach(), dout)
    for a, b in ((want["y"], y), (want["dx"], dx), (want["d_gates"], dg)):
        assert torch.allclose(a, b.detach(), rtol=1e-12, atol=1e-12)


def test_oracle_swiglu_at_its_codes():
    g, u, dh = (torch.randn(5, 150, generator=torch.Generator().manual_seed(i)).double() for i in range(3))
    h, dg, du, _, _ = oracle.swiglu(g, u, dh)
    kg, ku = (oracle.kept(t)[0].requires_grad_(True) for t in (g, u))
    a, b = torch.autograd.grad(torch.nn.functional.silu(kg) * ku, (kg, ku), dh)
    assert torch.allclose(h, torch.nn.functional.silu(g) * u) and torch.allclose(dg, a, rtol=1e-12, atol=1e-14) and torch.allclose(du, b, rtol=1e-12, atol=1e-14)
    for t, kt in ((g, kg), (u, ku)):
        for at in range(0, 150, 64):
            top = t[:, at:at + 64].abs().amax(1, keepdim=True)
            assert bool(((t - kt.detach())[:, at:at + 64].abs() <= top / 254 * (1 + 1e-12)).all())


def test_oracle_layer_is_the_definition():
    g = torch.Generator().manual_seed(3)
    x, wg = torch.randn(4, 8, generator=g).double(), torch.randn(3, 8, generator=g).double()
    w1, w3, w2 = (torch.randn(3, *s, generator=g).double() for s in ((6, 8), (6, 8), (8, 6)))
    out, weights, idx, _, _ = oracle.layer(x, wg, w1, w3, w2, 2)
    p = (x @ wg.t()).softmax(-1)
    top, want_idx = p.topk(2)
    want = sum((top[:, j] / top.sum(-1)).unsqueeze(-1) * torch.stack([w2[e] @ (torch.nn.functional.silu(w1[e] @ v) * (w3[e] @ v)) for e, v in zip(want_idx[:, j], x)]) for j in range(2))
    assert torch.equal(idx, want_idx) and torch.allclose(weights, top / top.sum(-1, keepdim=True)) and torch.allclose(out, want)
