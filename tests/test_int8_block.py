"""A block whose experts are to be held in 8 bits, on the host: what is refused before anything of the block changes,
and what a conversion leaves as it was."""
import pytest
import torch

import moe_distributed_training_amd as moe

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("match,kw", [
    ("float32", dict(dtype=F32)), ("multiples of 64", dict(hidden_size=96)), ("multiples of 64", dict(ffn_hidden_size=200, dtype=F16)),
    ("2\\^17", dict(hidden_size=1 << 17, num_experts=1, device="meta")), ("2\\^31", dict(hidden_size=64 * 1001, ffn_hidden_size=64 * 600, num_experts=1, device="meta")),
    ("lora_r = 0", dict(lora_r=8))])
def test_a_block_that_cannot_be_served_keeps_its_weights(match, kw):
    block = moe.ScatterMoEBlock(**{**dict(hidden_size=64, ffn_hidden_size=128, num_experts=2, dtype=BF16), **kw})
    before = {n: (p, p.dtype) for n, p in block.named_parameters()}
    with pytest.raises(ValueError, match=match):
        block.quantize_experts()
    assert not block.is_quantized and list(dict(block.named_buffers())) == []
    after = dict(block.named_parameters())
    assert list(after) == list(before) and all(after[n] is p and p.dtype == dt for n, (p, dt) in before.items())


def stand_in(dtype=BF16, E=2, f=128, d=64):
    """A block with codes and scales as quantize_experts() leaves them."""
    block = moe.ScatterMoEBlock(d, f, E, dtype=dtype)
    g = torch.Generator().manual_seed(0)
    for n, cols in (("w1", f), ("w2", d), ("w3", f)):
        delattr(block, n)
        block.register_buffer(n, torch.randint(-127, 128, (E, f, d), generator=g, dtype=torch.int8))
        block.register_buffer(n + "_scale", torch.rand(E, cols, generator=g) * 1e-3)
    assert block.is_quantized
    return block


@pytest.mark.parametrize("convert", [lambda m: m.to(BF16), lambda m: m.half(), lambda m: m.to("cpu", F16), lambda m: m.double(), lambda m: m.bfloat16()])
@pytest.mark.parametrize("inside", [False, True])
def test_a_conversion_does_not_round_the_scales(convert, inside):
    block = stand_in()
    before = {n: t.clone() for n, t in block.state_dict().items()}
    with pytest.raises(TypeError, match="float32"):
        convert(torch.nn.Sequential(block, torch.nn.Linear(4, 4)) if inside else block)
    assert all(t.dtype == before[n].dtype and torch.equal(t, before[n]) for n, t in block.state_dict().items())


def test_moves_and_conversions_that_keep_the_scales():
    import copy
    block = stand_in()
    before = {n: t.clone() for n, t in block.state_dict().items()}
    other = copy.deepcopy(block).to("cpu").cpu().requires_grad_(False).share_memory()
    assert all(torch.equal(t, before[n]) and t.dtype == before[n].dtype for n, t in other.state_dict().items())
    assert block.to("meta").w1_scale.dtype == F32 and block.to_empty(device="cpu").w2_scale.shape == (2, 64)
    block.load_state_dict(before)
    assert all(torch.equal(t, before[n]) for n, t in block.state_dict().items())
    plain = moe.ScatterMoEBlock(64, 128, 2, dtype=F32).to(BF16).half()          # blocks with their weights convert as ever
    assert plain.w1.dtype == F16


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_quantised_block_keeps_a_type_that_its_products_take(dtype):
    """An fp32 router would be served by nothing, and the way back would be refused for the scales' sake."""
    block = stand_in(dtype)
    for convert in (lambda m: m.float(), lambda m: m.to(F32)):
        with pytest.raises(TypeError, match="keeps its type"):
            convert(block)
    assert block.router.dtype == dtype and block.router.requires_grad and block.w2_scale.dtype == F32
