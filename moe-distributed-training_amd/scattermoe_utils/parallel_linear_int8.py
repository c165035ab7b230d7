"""Grouped linear over expert weights held in 8 bits: int8 codes with one fp32 scale for each expert's output column, and
activations turned into int8 codes with one scale for each row on the way.  No counterpart in the reference; the calling
convention is that of ``parallel_linear`` (scattermoe_utils/parallel_linear_lora.py:151-187 without adapters).

With cx, sx = codes and scales of the rows of x (``quantize_rows``) and cw, sw those of the weights
(``quantize_expert_weights``), row m of the sorted order, of expert e:

    y[out_row(m)][n] = sx[in_row(m)] * sw[e][n] * sum_k cx[in_row(m)][k] * cw[e][k][n]

The sum is exact (32-bit integers; fewer than 2^17 inputs), so it depends neither on the order of its terms nor on how the
work is divided.  The weights are frozen.  Gradients go straight through the rounding to codes, and are products of codes
too: with g_m = gate_m * dY_m * sw[e] and its codes cg, sg,

    dx[in_row(m)][k] += sg[m] * sum_n cg[m][n] * cw[e][k][n]
"""
from __future__ import annotations

from typing import Tuple

import torch

from .._lib import entry


def quantize_expert_weights(weights: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(E, K, N) weights, any strides -> (codes (E, K, N) int8, scales (E, N) fp32).  The scale of an output column is its
    largest magnitude / 127; a column that holds an infinity or a NaN gets the scale NaN.  The codes keep the orientation of
    the weights (contiguous along K, or along N) with rows padded to 16 bytes, which the products read in place."""
    codes, scales = entry("quantize_weights")(weights)
    return codes, scales


def parallel_linear_int8(inputs, expert_weights, weight_scales, k, sorted_expert_idxs, sorted_scattered_idxs, padded_block_idxs,
                         expert_offsets, gates=None, grouped_in=False, grouped_out=False):
    """``parallel_linear`` over 8-bit weights: inputs (rows, K) bf16, fp16 or fp32; expert_weights (E, K, N) int8 codes of
    any strides (codes whose rows are not contiguous and 16-byte aligned are copied within the call); weight_scales (E, N)
    fp32; the other arguments as in ``parallel_linear``.  Every assignment has to belong to an expert: rows of the result
    that no group covers are not written.  Gradients: of ``inputs`` (fewer than 2^17 output columns) and ``gates``."""
    return entry("linear_int8")(inputs, expert_weights, weight_scales, k, sorted_expert_idxs, sorted_scattered_idxs, expert_offsets, gates,
                                grouped_in, grouped_out)
