"""The expert-MLP caller of the MoE layer: w1 / w3 grouped GEMMs, SiLU * mul, w2 grouped GEMM, weighted combine.

Follows ``scattermoe_permute_and_compute`` of the reference (megablocks_utils/config_utils.py:99-185) and the weight
views it builds (``get_mlp_weights`` :28-35, ``get_mlp_weights_lora`` :37-61).  For bf16 tensors of Mixtral-like
shape the three projections run as two fused launches (dual-weight GEMM with SwiGLU epilogue, then w2) through
``moe_mlp_fwd`` / ``moe_mlp_bwd`` of libmoe_hip.so; everything else goes through the same three
``parallel_linear(_lora)`` calls the reference makes, which use the generic HIP kernels.  The sequences of library calls
and their autograd nodes are in csrc/torch_layer.cpp.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
import torch.nn as nn

from .._lib import entry, native, require_gpu
from ..scattermoe_utils.kernels import ops
from ..scattermoe_utils.parallel_experts import parallel_linear
from ..scattermoe_utils.parallel_linear_fp4 import quantize_expert_weights_fp4
from ..scattermoe_utils.parallel_linear_int8 import quantize_expert_weights
from ..scattermoe_utils.parallel_linear_lora import parallel_linear_lora


# ---------------------------------------------------------------------------------------------------------------
# weight views (reference config_utils.py:28-61)
# ---------------------------------------------------------------------------------------------------------------
def resolve_dtensor(t):
    """The local shard of a DTensor parameter, anything else unchanged (config_utils.py:32,58-59 strip the DTensor
    wrapper the same way before the kernels see the weights)."""
    return t.to_local() if hasattr(t, "to_local") else t


def get_mlp_weights(w: torch.Tensor, ffn_hidden_size: int, hidden_size: int, name: str = "w1") -> torch.Tensor:
    """Storage (E*ffn, hidden) -> the (E, K, N) view the kernels take: w1/w3 (E, hidden, ffn) K-contiguous,
    w2 (E, ffn, hidden) N-contiguous."""
    w = resolve_dtensor(w).view(-1, ffn_hidden_size, hidden_size)
    return w.permute(0, 2, 1) if name in ("w1", "w3") else w


def get_mlp_weights_lora(w: torch.Tensor, lora_A: torch.Tensor, lora_B: torch.Tensor, r: int,
                         ffn_hidden_size: int, hidden_size: int, name: str = "w1"):
    """Adapter storage of the reference (lora_A.weight kept transposed as (E*hidden, r), lora_B.weight (E*ffn, r),
    megablocks_utils/peft_utils.py:37-38,68-70) -> (W, A (E,K,r), B (E,r,N)) views, swapped for w2 (:51-56)."""
    W = get_mlp_weights(w, ffn_hidden_size, hidden_size, name)
    A = resolve_dtensor(lora_A).view(-1, hidden_size, r)
    B = resolve_dtensor(lora_B).view(-1, ffn_hidden_size, r).permute(0, 2, 1)
    if name == "w2":
        A, B = B.permute(0, 2, 1), A.permute(0, 2, 1)
    return W, A, B


class LoraViews(NamedTuple):
    a1: torch.Tensor
    b1: torch.Tensor
    a3: torch.Tensor
    b3: torch.Tensor
    a2: torch.Tensor
    b2: torch.Tensor


def fused_expert_mlp(x, w1, w2, w3, k, sorted_scattered_idxs, expert_offsets, lora: Optional[LoraViews] = None,
                     lora_alpha: float = 1.0, gates: Optional[torch.Tensor] = None, grouped_out: bool = False):
    """Expert MLP on expert-grouped assignments.  x (rows, d); w1, w2, w3 (E, f, d) in the reference's storage
    layout; ``k`` = fan-out of x rows (top_k, or 1 for pre-dispatched rows).  With ``gates`` (T, k) the k expert
    rows of each token are combined and (T, d) is returned; otherwise one row per assignment, in grouped order
    when ``grouped_out`` else at its flat position."""
    return entry("expert_mlp")(x, w1, w2, w3, k, sorted_scattered_idxs, expert_offsets, [] if lora is None else list(lora),
                               lora_alpha, gates, grouped_out)


class Int8ExpertWeights(NamedTuple):
    """Expert weights in 8 bits: codes (E, f, d) int8 in the reference's storage layout and, for each, the scales of its
    output columns: w1 and w3 (E, f), w2 (E, d)."""
    w1: torch.Tensor
    w1_scale: torch.Tensor
    w2: torch.Tensor
    w2_scale: torch.Tensor
    w3: torch.Tensor
    w3_scale: torch.Tensor

    @classmethod
    def quantize(cls, w1, w2, w3, ffn_hidden_size=None, hidden_size=None):
        """From bf16 / fp16 / fp32 weights (E, f, d), or in storage (E*f, d) with both sizes given."""
        out = []
        for name, w in (("w1", w1), ("w2", w2), ("w3", w3)):
            w = resolve_dtensor(w)
            if w.dim() == 2:
                w = w.view(-1, ffn_hidden_size, hidden_size)
            codes, scales = quantize_expert_weights(w if name == "w2" else w.transpose(1, 2))
            out += [(codes if name == "w2" else codes.transpose(1, 2)).contiguous(), scales]
        return cls(*out)


def fused_expert_mlp_int8(x, weights: Int8ExpertWeights, k, sorted_scattered_idxs, expert_offsets,
                          gates: Optional[torch.Tensor] = None, grouped_out: bool = False):
    """``fused_expert_mlp`` over 8-bit weights (frozen; no adapters): x (rows, d) bf16 or fp16, d and f multiples of 64, the
    other arguments and the result as there.  Both projections of a row work on one set of codes of it, the down projection
    on codes of h = silu(gate) * up.  Gradients: of x and ``gates``, straight through the rounding to codes; the gradient
    rows that meet weights are codes as well (dY times the gates and w2's scales; dgate and dup times their scales, one
    joint row); a gradient of x takes f below 2^16.  Every assignment has to belong to an expert."""
    return entry("expert_mlp_int8")(x, weights.w1, weights.w1_scale, weights.w2, weights.w2_scale, weights.w3, weights.w3_scale, k,
                                    sorted_scattered_idxs, expert_offsets, gates, grouped_out)


def swiglu_8bit(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """``silu(gate) * up`` of bf16, fp16 or fp32 tensors of one shape (any strides), keeping for the backward pass 8-bit codes of gate and up
    in place of the tensors: blocks of 64 columns with a scale each, 1.0625 bytes per value.  The result is that of the inputs as they
    are; the gradients are the formula's at the values that the codes stand for (off by at most 1/254 of their block's largest
    magnitude).  A block that holds an infinity or a NaN has NaN gradients."""
    return entry("swiglu_8bit")(gate, up)


class Fp4ExpertWeights(NamedTuple):
    """Expert weights in 4 bits (``quantize_expert_weights_fp4``): codes and scales, uint8, of w1 and w3 (E, f, d / 2) and (E, f, d / 32),
    and of w2 turned round, (E, d, f / 2) and (E, d, f / 32): every output's inputs lie side by side."""
    w1: torch.Tensor
    w1_scale: torch.Tensor
    w2: torch.Tensor
    w2_scale: torch.Tensor
    w3: torch.Tensor
    w3_scale: torch.Tensor

    @classmethod
    def quantize(cls, w1, w2, w3, ffn_hidden_size=None, hidden_size=None):
        """From bf16 / fp16 / fp32 weights (E, f, d), or in storage (E*f, d) with both sizes given."""
        out = []
        for name, w in (("w1", w1), ("w2", w2), ("w3", w3)):
            w = resolve_dtensor(w)
            if w.dim() == 2:
                w = w.view(-1, ffn_hidden_size, hidden_size)
            out += quantize_expert_weights_fp4(w if name == "w2" else w.transpose(1, 2))
        return cls(*out)


def fused_expert_mlp_fp4(x, weights: Fp4ExpertWeights, k, sorted_scattered_idxs, expert_offsets, gates: Optional[torch.Tensor] = None,
                         grouped_out: bool = False, keep_8bit: bool = False):
    """``fused_expert_mlp`` over 4-bit weights (frozen; no adapters): x (rows, d) bf16, fp16 or fp32, the other arguments and the result as
    there, one position for each of the rows' k assignments.  Gradients: of x and ``gates``.  ``keep_8bit``: the backward pass keeps
    gate and up as 8-bit codes (``swiglu_8bit``), 2.1 bytes per ffn value and assignment in place of 4 (fp32: 8).  Every assignment has to
    belong to an expert."""
    return entry("expert_mlp_fp4")(x, weights.w1, weights.w1_scale, weights.w2, weights.w2_scale, weights.w3, weights.w3_scale, k,
                                   sorted_scattered_idxs, expert_offsets, gates, grouped_out, keep_8bit)


def scattermoe_permute_and_compute(x, w1, w2, w3, ffn_hidden_size, hidden_size, top_k, bin_ids, indices, num_experts,
                                   lora_pointers=None, moe_expert_model_parallelism=True, expert_offsets=None,
                                   lora_views: Optional[LoraViews] = None, lora_alpha: float = 1.0, keep_8bit: bool = False):
    """Functional form of the reference caller (config_utils.py:99-185).

    x (rows, hidden); w1, w2, w3 storage (E*ffn, hidden); ``bin_ids`` / ``indices`` = sorted expert ids and sorted
    flat positions; ``lora_pointers[name] = (A.weight, B.weight, r, alpha, hidden, ffn)`` as peft_utils.py:127-132
    (or ``lora_views`` / ``lora_alpha``: the six factor views already in (E, K, r) / (E, r, N) form).
    Expert-parallel mode treats x as pre-dispatched rows (fan-out 1) and scatters the output back to ``indices``;
    otherwise the fan-out is top_k and the output stays in grouped order (the caller's ops.scatter combines it).  ``keep_8bit``: gate
    and up kept for the backward pass as 8-bit codes (``swiglu_8bit``), 4.1 bytes per ffn value and assignment in place of 6; through the
    three projections one by one, which makes a step of wide experts 7 % longer (15 % with adapters), of narrow ones 13 % (33 %)."""
    with torch.no_grad():
        if expert_offsets is None:
            expert_offsets = ops.expert_offsets_from_sorted(bin_ids, num_experts)
    fan = 1 if moe_expert_model_parallelism else top_k
    grouped_out = not moe_expert_model_parallelism
    W = {n: w.view(-1, ffn_hidden_size, hidden_size) for n, w in (("w1", w1), ("w2", w2), ("w3", w3))}
    lora = None
    alpha = 1.0
    if lora_pointers is not None:
        v = {}
        for n in ("w1", "w2", "w3"):
            A, B, r, alpha, hs, fs = lora_pointers[n]
            _, v["a" + n[1]], v["b" + n[1]] = get_mlp_weights_lora(W[n], A, B, r, fs, hs, n)
        lora = LoraViews(v["a1"], v["b1"], v["a3"], v["b3"], v["a2"], v["b2"])
    elif lora_views is not None:
        lora, alpha = lora_views, lora_alpha
    if not keep_8bit and native.mlp_fast_path(x, W["w1"], W["w2"], W["w3"], [] if lora is None else list(lora)):
        return fused_expert_mlp(x, W["w1"], W["w2"], W["w3"], fan, indices, expert_offsets, lora, alpha, None, grouped_out)
    # generic route: the reference's three calls (:127-166)
    def proj(inp, name, kk, gin, gout):
        Wv = get_mlp_weights(W[name], ffn_hidden_size, hidden_size, name)
        if lora is None:
            return parallel_linear(inp, Wv, kk, bin_ids, indices, None, expert_offsets, None, gin, gout)
        a, b = getattr(lora, "a" + name[1]), getattr(lora, "b" + name[1])
        return parallel_linear_lora(inp, Wv, a, b, a.size(2), alpha, kk, bin_ids, indices, None, expert_offsets, None,
                                    gin, gout)
    h1 = proj(x, "w1", fan, False, True)
    h3 = proj(x, "w3", fan, False, True)
    h = swiglu_8bit(h1, h3) if keep_8bit else entry("swiglu")(h1, h3)
    return proj(h, "w2", 1, True, grouped_out)


# ---------------------------------------------------------------------------------------------------------------
# whole layer: router -> sort -> expert MLP -> weighted combine, one autograd node
# ---------------------------------------------------------------------------------------------------------------
def moe_layer_forward(x, wg, w1, w2, w3, top_k=2, lora: Optional[LoraViews] = None, lora_alpha: float = 1.0,
                      normalize: bool = True):
    """x (T, d) bf16 -> (out (T, d), expert_weights (T, k) fp32, expert_indices (T, k) int32).
    wg (E, d) router weight; w1, w2, w3 (E, f, d) expert weights in the reference's storage layout."""
    return _layer(x, wg, w1, w2, w3, w1.size(0), w1.size(1), top_k, [] if lora is None else list(lora), lora_alpha, normalize, False)


def _empty_layer(x, wg, weights, top_k):
    """An empty batch routes nothing: empty outputs, and backward leaves every parameter's grad unset."""
    require_gpu(x, wg, *weights)
    return (x.clone(), torch.zeros((0, top_k), dtype=torch.float32, device=x.device),
            torch.zeros((0, top_k), dtype=torch.int32, device=x.device))


def _layer(x, wg, w1, w2, w3, E, f, top_k, lora, lora_alpha, normalize, storage):
    if x.size(0) == 0:
        return _empty_layer(x, wg, (w1, w2, w3), top_k)
    return entry("layer")(x, wg, w1, w2, w3, E, f, top_k, lora, lora_alpha, bool(normalize), storage)


def moe_layer_forward_int8(x, wg, weights: Int8ExpertWeights, top_k=2, normalize: bool = True):
    """``moe_layer_forward`` over 8-bit expert weights: x (T, d) bf16 or fp16 -> (out (T, d), expert_weights (T, k) fp32,
    expert_indices (T, k) int32).  Gradients: of x and the router weight wg."""
    if x.size(0) == 0:
        return _empty_layer(x, wg, weights, top_k)
    return entry("layer_int8")(x, wg, weights.w1, weights.w1_scale, weights.w2, weights.w2_scale, weights.w3, weights.w3_scale, top_k,
                               bool(normalize))


def moe_layer_forward_fp4(x, wg, weights: Fp4ExpertWeights, top_k=2, normalize: bool = True, keep_8bit: bool = False):
    """``moe_layer_forward`` over 4-bit expert weights: x (T, d) bf16, fp16 or fp32 -> (out (T, d), expert_weights (T, k) fp32,
    expert_indices (T, k) int32).  Up to 16 bf16 or fp16 tokens of at most 256 experts and 16 per token, d and f multiples of 64, without
    gradients run as two launches, with fewer roundings on the way; they rank experts as the other launches do, by fp32 scores, whose logits
    are sums in another order.  Weights at odd addresses or strides are copied in every call.  Gradients: of x and the router weight wg;
    ``keep_8bit`` as in ``fused_expert_mlp_fp4``."""
    if x.size(0) == 0:
        return _empty_layer(x, wg, weights, top_k)
    return entry("layer_fp4")(x, wg, weights.w1, weights.w1_scale, weights.w2, weights.w2_scale, weights.w3, weights.w3_scale, top_k,
                              bool(normalize), bool(keep_8bit))


def moe_layer_decode(x, wg, w1, w2, w3, top_k=2, normalize: bool = True):
    """``moe_layer_forward`` for the tokens of a generation step, in two launches and without gradients: x (T, d), T up to 16, wg (E, d) and
    w1, w2, w3 (E, f, d), all bf16 or all fp16, E up to 256, top_k up to 16, d and f multiples of 64 -> (out (T, d), expert_weights (T, k) fp32,
    expert_indices (T, k) int32).  The weights of a chosen expert are read once, however many tokens chose it.  Weights that are not
    contiguous, or start at no multiple of 16 bytes, are copied whole in every call, all experts: lay them out once.  Experts are ranked by
    their fp32 scores as in ``moe_layer_forward``; the result differs from its by roundings (the interim of the two projections keeps
    2^-17 of itself in bf16, 2^-23 in fp16, there 2^-8 and 2^-11), and experts whose logits differ by less than the rounding of a sum may be
    ranked either way.  Narrow experts take down to two thirds of its time, wide ones the same within 4 % (both read the weights at the
    memory's rate)."""
    return entry("layer_decode")(x, wg, w1, w2, w3, top_k, bool(normalize))


class ScatterMoEBlock(nn.Module):
    """Drop-in for a Mixtral sparse-MoE block built the way the reference builds it: router weight (E, d), expert
    weights w1, w2, w3 stored (E*f, d) (megablocks_utils/sparse_mlp2.py:22-36, HF w2 transposed on load,
    shard_moe_utils.py:153-157), optional LoRA factors stored as peft_utils.py:37-38,68-70 does.  Returns
    ``(hidden, None)`` like the patched ParallelMLP.forward (config_utils.py:75-92); with ``bias=True`` the block owns an
    output bias (megablocks' ``ParallelMLP.bias``) and follows that method's bias branch (config_utils.py:80-84):
    ``(hidden, bias)`` when ``return_bias`` is set, otherwise the single tensor ``hidden + bias``."""

    def __init__(self, hidden_size, ffn_hidden_size, num_experts, top_k=2, lora_r=0, lora_alpha=16.0,
                 dtype=torch.bfloat16, device=None, bias=False, return_bias=False):
        super().__init__()
        self.return_bias = return_bias
        self.keep_8bit = False
        self.bias = nn.Parameter(torch.zeros(hidden_size, dtype=dtype, device=device)) if bias else None
        self.hidden_size, self.ffn_hidden_size = hidden_size, ffn_hidden_size
        self.num_experts, self.top_k, self.lora_r, self.lora_alpha = num_experts, top_k, lora_r, lora_alpha
        kw = dict(dtype=dtype, device=device)
        self.router = nn.Parameter(torch.empty(num_experts, hidden_size, **kw))
        self.w1 = nn.Parameter(torch.empty(num_experts * ffn_hidden_size, hidden_size, **kw))
        self.w2 = nn.Parameter(torch.empty(num_experts * ffn_hidden_size, hidden_size, **kw))
        self.w3 = nn.Parameter(torch.empty(num_experts * ffn_hidden_size, hidden_size, **kw))
        for p in (self.router, self.w1, self.w2, self.w3):
            nn.init.normal_(p, std=0.02)
        if lora_r > 0:
            for n in ("w1", "w2", "w3"):
                a = nn.Parameter(torch.empty(num_experts * hidden_size, lora_r, **kw))
                b = nn.Parameter(torch.zeros(num_experts * ffn_hidden_size, lora_r, **kw))
                nn.init.normal_(a, std=0.02)
                self.register_parameter(f"lora_A_{n}", a)
                self.register_parameter(f"lora_B_{n}", b)
            for p in (self.router, self.w1, self.w2, self.w3) + (() if self.bias is None else (self.bias,)):
                p.requires_grad_(False)

    def lora_views(self) -> Optional[LoraViews]:
        if self.lora_r == 0:
            return None
        v = {}
        for n in ("w1", "w2", "w3"):
            _, a, b = get_mlp_weights_lora(getattr(self, n), getattr(self, f"lora_A_{n}"), getattr(self, f"lora_B_{n}"),
                                           self.lora_r, self.ffn_hidden_size, self.hidden_size, n)
            v["a" + n[1]], v["b" + n[1]] = a, b
        return LoraViews(v["a1"], v["b1"], v["a3"], v["b3"], v["a2"], v["b2"])

    def quantize_experts(self, bits: int = 8, keep_8bit: bool = False) -> "ScatterMoEBlock":
        """Puts codes in the place of the expert weights, for serving and for training what lies before and around them.

        ``bits`` 8: w1, w2, w3 become int8 buffers (E, f, d) with fp32 buffers ``w1_scale``, ``w2_scale``, ``w3_scale`` of their output
        columns, and ``forward`` takes the products over them (bf16 or fp16 hidden states, sizes that are multiples of 64).  The router
        keeps its type, and the block from then on: a conversion that would round the scales is refused.
        ``bits`` 4: uint8 buffers of ``Fp4ExpertWeights``; a batch of up to 16 tokens without gradients runs as two launches;
        ``keep_8bit`` as in ``fused_expert_mlp_fp4``.

        Not for a block with adapters: its factors are trained against the weights as they are.  A block that the products could not
        serve is refused and keeps its weights."""
        if bits not in (4, 8):
            raise ValueError(f"expert weights are held in 8 or 4 bits, not {bits}")
        if keep_8bit and bits != 4:
            raise ValueError("keep_8bit goes with experts in 4 bits: the products over 8-bit weights keep interims of their own")
        if self.lora_r > 0:
            raise ValueError("a block with adapters keeps its expert weights: quantize_experts() takes blocks with lora_r = 0")
        if self.is_quantized:
            if bits != self.expert_bits:
                raise ValueError(f"the experts are held in {self.expert_bits} bits already; their weights are gone")
            self.keep_8bit = bool(keep_8bit)
            return self
        d, f = self.hidden_size, self.ffn_hidden_size
        if bits == 4:
            if self.router.dtype not in (torch.bfloat16, torch.float16, torch.float32):
                raise ValueError(f"the expert MLP over 4-bit weights takes bf16, fp16 or fp32 hidden states, this block's are {self.router.dtype}")
            if max(d, f) > 2 ** 20 or d * f >= 2 ** 31:
                raise ValueError(f"the expert MLP over 4-bit weights takes sizes up to 2^20, together below 2^31, not hidden size {d} and ffn size {f}")
            q = Fp4ExpertWeights.quantize(self.w1, self.w2, self.w3, f, d)
        else:
            if self.router.dtype not in (torch.bfloat16, torch.float16):
                raise ValueError(f"the expert MLP over 8-bit weights takes bf16 or fp16 hidden states, this block's are {self.router.dtype}: "
                                 "convert the block first")
            if d % 64 or f % 64 or max(d, f) >= 2 ** 17 or d * f >= 2 ** (31 if d % 128 or f % 128 else 32) - 16:
                raise ValueError(f"the expert MLP over 8-bit weights takes sizes that are multiples of 64, below 2^17 and together below 2^32 (2^31 "
                                 f"where one is no multiple of 128), not hidden size {d} and ffn size {f}")
            q = Int8ExpertWeights.quantize(self.w1, self.w2, self.w3, f, d)
        for name, t in q._asdict().items():
            if hasattr(self, name):
                delattr(self, name)
            self.register_buffer(name, t)
        self.keep_8bit = bool(keep_8bit)
        return self

    @property
    def expert_bits(self) -> int:
        """Bits of an expert weight: 4 or 8 after ``quantize_experts``, otherwise those of its type."""
        return {torch.uint8: 4, torch.int8: 8}.get(self.w1.dtype) or torch.finfo(self.w1.dtype).bits

    @property
    def is_quantized(self) -> bool:
        return self.w1.dtype in (torch.int8, torch.uint8)

    def _apply(self, fn, *args, **kw):
        # (what ``to``, ``half``, ``cuda`` and the like go through, also those of a module around this one; 4-bit weights have no type to lose)
        if self.w1.dtype == torch.int8 and any(fn(t.detach()[:0]).dtype != t.dtype for t in (self.w1_scale, self.router)):
            raise TypeError("a block with experts in 8 bits keeps its type, and its scales stay float32: choose the type before quantize_experts()")
        return super()._apply(fn, *args, **kw)

    def _weights(self, kind):
        return kind(*(getattr(self, n) for n in kind._fields))

    def decode(self, hidden_states: torch.Tensor):
        """``forward`` for the tokens of a generation step, without gradients: up to 16 of them through ``moe_layer_decode`` (two launches;
        a block without adapters, bf16 or fp16 weights or weights in 4 bits).  Returns as ``forward`` does."""
        if self.lora_r > 0:
            raise ValueError("decode() takes blocks without adapters (lora_r = 0): use forward()")
        with torch.no_grad():
            if self.is_quantized:
                return self.forward(hidden_states)
            x = hidden_states.reshape(-1, hidden_states.shape[-1])
            w = [resolve_dtensor(t).view(self.num_experts, self.ffn_hidden_size, self.hidden_size) for t in (self.w1, self.w2, self.w3)]
            return self._returned(moe_layer_decode(x, resolve_dtensor(self.router), *w, self.top_k)[0].view(hidden_states.shape))

    def forward(self, hidden_states: torch.Tensor):
        shape = hidden_states.shape
        x = hidden_states.reshape(-1, shape[-1])
        E, f = self.num_experts, self.ffn_hidden_size
        lora = []
        if self.lora_r > 0:   # the factors in their storage, in the order a1, b1, a3, b3, a2, b2 (w2's are swapped, see lora_views)
            lora = [resolve_dtensor(t) for t in (self.lora_A_w1, self.lora_B_w1, self.lora_A_w3, self.lora_B_w3, self.lora_B_w2, self.lora_A_w2)]
        if self.w1.dtype == torch.int8:
            out = moe_layer_forward_int8(x, resolve_dtensor(self.router), self._weights(Int8ExpertWeights), self.top_k)[0]
        elif self.w1.dtype == torch.uint8:
            out = moe_layer_forward_fp4(x, resolve_dtensor(self.router), self._weights(Fp4ExpertWeights), self.top_k, keep_8bit=self.keep_8bit)[0]
        else:
            out = _layer(x, resolve_dtensor(self.router), resolve_dtensor(self.w1), resolve_dtensor(self.w2), resolve_dtensor(self.w3), E, f,
                         self.top_k, lora, self.lora_alpha, True, True)[0]
        return self._returned(out.view(shape))

    def _returned(self, out):
        if self.bias is not None:
            if self.return_bias:
                return out, self.bias
            return out + self.bias
        return out, None
