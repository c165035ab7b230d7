"""Grouped linear over expert weights held in 4 bits: codes of one sign, two exponent and one mantissa bit (0, 0.5, 1, 1.5, 2,
3, 4, 6) and one power of two for each 32 consecutive inputs of an expert's output column.  No counterpart in the reference;
the calling convention is that of ``parallel_linear`` (scattermoe_utils/parallel_linear_lora.py:151-187 without adapters).

    W[e][n][k] = code[e][n][k] * 2^(scale[e][n][k // 32] - 127)
    y[out_row(m)][n] = sum_k x[in_row(m)][k] * W[e][n][k]

Activations stay as they are: the products are those of a 16-bit (or 32-bit) linear over the weights that the codes stand for,
which bf16 and fp32 hold exactly.  The weights are frozen; dx[in_row(m)][k] += gate_m * sum_n dY[m][n] * W[e][n][k].
"""
from __future__ import annotations

from typing import Tuple

import torch

from .._lib import entry


def quantize_expert_weights_fp4(weights: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(E, K, N) weights, any strides -> (codes (E, N, ceil(K / 32) * 16) uint8, scales (E, N, ceil(K / 32)) uint8).  Byte b of a
    column's codes holds inputs 2b (lower half) and 2b + 1; zeros behind K.  The power of two of a group is the least that leaves its
    largest magnitude at 7 units or below, and every weight becomes the nearest code, the even one of two.  A group of zeros has the
    scale 0 (2^-127), one that holds an infinity or a NaN the scale 255, which stands for NaN, and codes 0."""
    codes, scales = entry("quantize_weights_fp4")(weights)
    return codes, scales


def parallel_linear_fp4(inputs, expert_codes, weight_scales, k, sorted_expert_idxs, sorted_scattered_idxs, padded_block_idxs,
                        expert_offsets, gates=None, grouped_in=False, grouped_out=False):
    """``parallel_linear`` over 4-bit weights: inputs (rows, K) bf16, fp16 or fp32; expert_codes and weight_scales as
    ``quantize_expert_weights_fp4`` returns them, of any strides (codes whose rows are not contiguous and 16-byte aligned are copied
    within the call, and with 16-bit inputs the scales where ceil(K / 32) or a stride is no multiple of 4); the other arguments as in ``parallel_linear``.  With fp16 inputs the weights are numbers of fp16: scales from 104
    to 140 are exact, beyond them weights round, or overflow to infinity.  Every assignment has to belong to an expert: rows of the
    result that no group covers are not written.  Gradients: of ``inputs`` and ``gates``."""
    return entry("linear_fp4")(inputs, expert_codes, weight_scales, k, sorted_expert_idxs, sorted_scattered_idxs, expert_offsets, gates, grouped_in,
                               grouped_out)
