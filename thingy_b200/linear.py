"""A linear layer in 8 bits, forward and backward: casts and block-scaled products.

``fp8_linear(x, weight)`` is ``x @ weight.T`` computed on e4m3 codes, under
autograd: x and the incoming gradient are cast in 1 x 128 groups along both
axes, the weight in 128 x 128 blocks, and the three products of a training
step run through ``fp8_block_gemm``. The reference stops at the quantizer
(src/cutie/rms_norm/bench.py:4-7); this is the layer its codes are made for.
"""

from __future__ import annotations

import torch

from .fp8_utils import per_block_cast_to_fp8, per_token_cast_to_fp8, two_way_cast_to_fp8
from .gemm import fp8_block_gemm


class FP8Linear(torch.autograd.Function):
    """(x [M, K], weight [N, K], weight_fp8 or None) -> y [M, N], all bf16.

    The straight-through gradients of a layer whose operands are quantized:
    dx = q(dy) q(w), dw = q(dy)^T q(x), with x and dy quantized along the
    token axis for dw. dw has the weight's dtype (bf16 or fp32).
    """

    @staticmethod
    def forward(ctx, x, weight, weight_fp8=None):
        need_dx, need_dw = ctx.needs_input_grad[:2]
        if weight_fp8 is None:
            w = weight.to(torch.bfloat16)
            weight_fp8 = per_block_cast_to_fp8(w, transposed=True) if need_dx \
                else (*per_block_cast_to_fp8(w), None, None)
        wq, ws, wqt, wst = weight_fp8
        if need_dw:
            q, s, qt, st = two_way_cast_to_fp8(x)
        elif x.shape[-1] % 16 == 0:
            (q, s), qt, st = per_token_cast_to_fp8(x, False), None, None
        else:  # rows of codes off the 16-byte boundaries that the product needs
            q, s, _, _ = two_way_cast_to_fp8(x)
            qt = st = None
        ctx.save_for_backward(qt, st, wqt, wst)
        ctx.weight_dtype = weight.dtype
        return fp8_block_gemm(q, s, wq, ws)

    @staticmethod
    def backward(ctx, dy):
        qt, st, wqt, wst = ctx.saved_tensors
        need_dx, need_dw = ctx.needs_input_grad[:2]
        dx = dw = None
        q, s, dqt, dst = two_way_cast_to_fp8(dy.contiguous())
        if need_dx:
            if wqt is None:
                raise ValueError("weight_fp8 has no transposed codes: make it with "
                                 "per_block_cast_to_fp8(weight, transposed=True)")
            dx = fp8_block_gemm(q, s, wqt, wst)
        if need_dw:
            dw = fp8_block_gemm(dqt, dst, qt, st, out_dtype=ctx.weight_dtype)
        return dx, dw, None


def fp8_linear(x: torch.Tensor, weight: torch.Tensor, weight_fp8=None) -> torch.Tensor:
    """``x @ weight.T`` on e4m3 codes with fp32 sums, bf16 out, differentiable in x and weight.

    x: bf16 [..., K]; weight: bf16 or fp32 [N, K]; K and N multiples of 8.
    ``weight_fp8``: (q, s, qt, st) of ``per_block_cast_to_fp8(weight,
    transposed=True)`` where the caller casts the weight once for several
    calls (an optimizer step, inference: there (q, s, None, None) does);
    without it the weight is cast in the call. Runs on the current stream.
    """
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} must be [..., K] and [N, K]")
    if x.dtype != torch.bfloat16:
        raise ValueError(f"x must be bfloat16, got {x.dtype}")
    if weight.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"weight must be bfloat16 or float32, got {weight.dtype}")
    if weight.shape[0] % 8 != 0 or weight.shape[1] % 8 != 0:
        raise ValueError(f"weight's sizes must be multiples of 8, got {tuple(weight.shape)}")
    y = FP8Linear.apply(x.reshape(-1, x.shape[-1]), weight, weight_fp8)
    return y.reshape(*x.shape[:-1], weight.shape[0])
