"""A linear layer in 8 bits, forward and backward: casts and block-scaled products.

``fp8_linear(x, weight)`` is ``x @ weight.T`` computed on e4m3 codes, under
autograd: x and the incoming gradient are cast in 1 x 128 groups along both
axes, the weight in 128 x 128 blocks, and the three products of a training
step run through the block-scaled GEMM (``fp8_block_gemm``). The reference
stops at the quantizer (src/cutie/rms_norm/bench.py:4-7); this is the layer
its codes are made for.
"""

from __future__ import annotations

import torch

from .ops import require_binding


def fp8_linear(x: torch.Tensor, weight: torch.Tensor, weight_fp8=None) -> torch.Tensor:
    """``x @ weight.T`` on e4m3 codes with fp32 sums, bf16 out, differentiable in x and weight.

    x: bf16 [..., K]; weight: bf16 or fp32 [N, K] (fp32 is rounded to bf16
    first, then to e4m3); K and N multiples of 8.
    Both, and y's gradient, may have any strides; a matrix whose rows are not
    dense and on 16-byte boundaries is copied first.
    ``weight_fp8``: (q, s, qt, st) of ``per_block_cast_to_fp8(weight,
    transposed=True)`` where the caller casts the weight once for several
    calls (an optimizer step, inference: there (q, s, None, None) does);
    without it the weight is cast in the call. The gradients are the
    straight-through ones of quantized operands: dx = q(dy) q(w), dw = q(dy)^T
    q(x), with x and dy quantized along the token axis for dw; dw has the
    weight's dtype. x and the weight are cast with the quantizers' least scale
    of 1e-4; a group of dy that is below 1e-4 throughout has a scale of its own
    (``two_way_cast_to_fp8(..., gradient=True)``), so no gradient is too small.
    Runs on the current stream.
    """
    wq, ws, wqt, wst = (None, None, None, None) if weight_fp8 is None else weight_fp8
    return require_binding().fp8_linear(x, weight, wq, ws, wqt, wst)
