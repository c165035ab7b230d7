"""A block whose experts are to be held in 8 bits, on the host: what is refused before anything of the block changes."""
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
