"""thingy_b200 — B200-native (sm_100a) residual-add + RMSNorm + FP8 quantization.

Drop-in host API for the reference's hot path (S1ro1/thingy, package
``cutie``):

    RMSNorm, rms_norm, rms_norm_on_stream   <- src/cutie/rms_norm/rms_norm.py
    residual_rms_norm_fp8                   <- residual_rms_norm_fp8_reference,
                                               src/cutie/rms_norm/bench.py:83-100
    per_token_cast_to_fp8(_triton)          <- src/cutie/vendor/prime_rl/fp8_utils.py:63-89
    rms_norm_fp8                            general form (per-token / 1xG / MXFP8,
                                               fp32 / pow2 / e8m0 scales, layouts)
    rms_norm_fp8_backward, ResidualRMSNormFP8
                                            backward (no counterpart in the reference):
                                               the gradients autograd gives its forward

    per_block_cast_to_fp8, two_way_cast_to_fp8, fp8_block_gemm, fp8_linear
                                            what follows the quantizer (no counterpart):
                                               weight and two-way casts, the product with a
                                               scale a block of 128, a linear layer with its
                                               gradients
    moe_fp8, quantize_experts               a mixture-of-experts layer for few tokens in one
                                               kernel, forward only (no counterpart)
    moe_sort, moe_permute, moe_combine      tokens sorted by expert and back, with weights
                                               applied, and the gradients (no counterpart)
    fp8_grouped_gemm, fp8_grouped_linear    the experts' products on sorted rows, and their
                                               linear layer with its gradients (no counterpart)
    adamw_step, adamw_state, AdamW          an optimizer step over many tensors in one launch,
                                               states in 32 bits or in 8 (no counterpart)

Every op runs hand-written CUDA from ``lib/libcutie_b200.so`` through the C
ABI in ``include/cutie.h``; there is no CPU or PyTorch fallback.
"""

from .backward import ResidualRMSNormFP8, rms_norm_fp8_backward
from .dispatch import MoePlan, moe_combine, moe_permute, moe_plan_rows, moe_sort
from .fp8_utils import (per_block_cast_to_fp8, per_token_cast_to_fp8, per_token_cast_to_fp8_triton,
                        two_way_cast_to_fp8)
from .fused import empty_scale, residual_rms_norm_fp8, rms_norm_fp8
from .gemm import fp8_block_gemm, fp8_grouped_gemm
from .layouts import mx_swizzle, mx_swizzle_offset, mx_swizzled_size, mx_unswizzle
from .linear import fp8_grouped_linear, fp8_linear
from .moe import clear_moe_workspaces, moe_fp8, moe_workspace, quantize_experts
from .optim import AdamW, adamw_state, adamw_step
from .rms_norm import RMSNorm, rms_norm, rms_norm_on_stream

__all__ = [
    "AdamW",
    "MoePlan",
    "RMSNorm",
    "ResidualRMSNormFP8",
    "adamw_state",
    "adamw_step",
    "clear_moe_workspaces",
    "empty_scale",
    "fp8_block_gemm",
    "fp8_grouped_gemm",
    "fp8_grouped_linear",
    "fp8_linear",
    "moe_combine",
    "moe_fp8",
    "moe_permute",
    "moe_plan_rows",
    "moe_sort",
    "moe_workspace",
    "mx_swizzle",
    "mx_swizzle_offset",
    "mx_swizzled_size",
    "mx_unswizzle",
    "per_block_cast_to_fp8",
    "per_token_cast_to_fp8",
    "per_token_cast_to_fp8_triton",
    "quantize_experts",
    "residual_rms_norm_fp8",
    "rms_norm",
    "rms_norm_fp8",
    "rms_norm_fp8_backward",
    "rms_norm_on_stream",
    "two_way_cast_to_fp8",
]
