"""torch.library ops so torch.compile(fullgraph=True) regions can call the path.

``thingy_b200::per_token_fp8_quant`` has the schema of the reference's
``cutie::per_token_fp8_quant`` (src/cutie/rms_norm/bench.py:68-80):
bf16 [M, H] -> (e4m3 [M, H], fp32 [M, ceil(H / 128)]), with a fake (meta)
implementation for tracing. ``thingy_b200::residual_rms_norm_fp8`` is the
whole fused contract (bench.py:10-11): (q, scale, residual_out, normalized).

What follows the quantizer has ops too: ``thingy_b200::per_block_cast_to_fp8``,
``thingy_b200::two_way_cast_to_fp8``, ``thingy_b200::fp8_block_gemm`` and
``thingy_b200::moe_fp8``; for many tokens ``thingy_b200::moe_sort``,
``thingy_b200::moe_permute``, ``thingy_b200::fp8_grouped_gemm`` (a plan with align 128)
and ``thingy_b200::moe_combine``. They are forward only.

Importing this module also registers ``cutie::per_token_fp8_quant`` itself,
the name the reference's callers use (``torch.ops.cutie.per_token_fp8_quant``),
backed by this library, unless some module (the reference's own bench.py,
say) has already defined an op of that name: then that one is left in place
and ``REFERENCE_NAMESPACE_OP`` is False. The standalone RMSNorm ops
(``thingy_b200::rms_norm``, ``thingy_b200::rms_norm_out``) are registered by
``thingy_b200.rms_norm``.
"""

from __future__ import annotations

import torch

from .dispatch import MoePlan, moe_combine, moe_permute
from .fp8_utils import per_token_cast_to_fp8
from .fp8_utils import per_block_cast_to_fp8, two_way_cast_to_fp8
from .fused import residual_rms_norm_fp8
from .gemm import fp8_block_gemm, fp8_grouped_gemm
from .moe import moe_fp8
from .ops import require_binding

GROUP_SIZE = 128


@torch.library.custom_op("thingy_b200::per_token_fp8_quant", mutates_args=())
def quantize_fp8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return per_token_cast_to_fp8(x, use_ue8m0=False)


@quantize_fp8.register_fake
def _quantize_fp8_fake(x):
    return (
        torch.empty_like(x, dtype=torch.float8_e4m3fn),
        x.new_empty((x.shape[0], -(-x.shape[1] // GROUP_SIZE)), dtype=torch.float32),
    )


@torch.library.custom_op("thingy_b200::residual_rms_norm_fp8", mutates_args=())
def residual_rms_norm_fp8_op(
    x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return residual_rms_norm_fp8(x, residual, weight, eps)


@residual_rms_norm_fp8_op.register_fake
def _residual_rms_norm_fp8_fake(x, residual, weight, eps):
    return (
        torch.empty_like(x, dtype=torch.float8_e4m3fn),
        x.new_empty((x.shape[0], -(-x.shape[1] // GROUP_SIZE)), dtype=torch.float32),
        torch.empty_like(x),
        torch.empty_like(x),
    )


def _codes(x, rows: int, cols: int) -> torch.Tensor:
    return x.new_empty_strided((rows, cols), (-(-cols // 16) * 16, 1), dtype=torch.float8_e4m3fn)


@torch.library.custom_op("thingy_b200::per_block_cast_to_fp8", mutates_args=())
def per_block_cast_op(w: torch.Tensor, use_ue8m0: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return per_block_cast_to_fp8(w, use_ue8m0, transposed=True)


@per_block_cast_op.register_fake
def _per_block_cast_fake(w, use_ue8m0):
    R, C = w.shape
    GR, GC = -(-R // GROUP_SIZE), -(-C // GROUP_SIZE)
    return (_codes(w, R, C), w.new_empty((GR, GC), dtype=torch.float32),
            _codes(w, C, R), w.new_empty((GC, GR), dtype=torch.float32))


@torch.library.custom_op("thingy_b200::two_way_cast_to_fp8", mutates_args=())
def two_way_cast_op(x: torch.Tensor, use_ue8m0: bool, gradient: bool = False) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return two_way_cast_to_fp8(x, use_ue8m0, gradient)


@two_way_cast_op.register_fake
def _two_way_cast_fake(x, use_ue8m0, gradient=False):
    R, C = x.shape
    GR, GC = -(-R // GROUP_SIZE), -(-C // GROUP_SIZE)
    return (_codes(x, R, C), x.new_empty_strided((R, GC), (1, R), dtype=torch.float32),
            _codes(x, C, R), x.new_empty_strided((C, GR), (1, C), dtype=torch.float32))


@torch.library.custom_op("thingy_b200::fp8_block_gemm", mutates_args=())
def fp8_block_gemm_op(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
                      fp32_out: bool) -> torch.Tensor:
    return fp8_block_gemm(a, a_scale, b, b_scale,
                          out_dtype=torch.float32 if fp32_out else torch.bfloat16)


@fp8_block_gemm_op.register_fake
def _fp8_block_gemm_fake(a, a_scale, b, b_scale, fp32_out):
    return a.new_empty((a.shape[0], b.shape[0]), dtype=torch.float32 if fp32_out else torch.bfloat16)


@torch.library.custom_op("thingy_b200::moe_fp8", mutates_args=())
def moe_fp8_op(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor, router: torch.Tensor,
               w13: torch.Tensor, w13_scale: torch.Tensor, w2: torch.Tensor, w2_scale: torch.Tensor,
               top_k: int, scoring: str, renormalize: bool, routed_scale: float,
               bias: torch.Tensor | None) -> torch.Tensor:
    return moe_fp8(x, q, scale, router, w13, w13_scale, w2, w2_scale, top_k=top_k, scoring=scoring,
                   renormalize=renormalize, routed_scale=routed_scale, bias=bias)


@moe_fp8_op.register_fake
def _moe_fp8_fake(x, q, scale, router, w13, w13_scale, w2, w2_scale, top_k, scoring, renormalize,
                  routed_scale, bias):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


@torch.library.custom_op("thingy_b200::moe_sort", mutates_args=())
def moe_sort_op(topk_ids: torch.Tensor, num_experts: int, align: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return require_binding().moe_sort(topk_ids, num_experts, align, True)


@moe_sort_op.register_fake
def _moe_sort_fake(topk_ids, num_experts, align):
    T, k = topk_ids.shape
    rows = (T * k + min(num_experts, T * k) * (align - 1)) // align * align
    return (topk_ids.new_empty((rows,), dtype=torch.int32), topk_ids.new_empty((T, k), dtype=torch.int32),
            topk_ids.new_empty((num_experts + 1,), dtype=torch.int32), topk_ids.new_empty((num_experts,), dtype=torch.int32))


@torch.library.custom_op("thingy_b200::moe_permute", mutates_args=())
def moe_permute_op(x: torch.Tensor, sources: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    return moe_permute(x, MoePlan(sources, positions, None, None, 1))


@moe_permute_op.register_fake
def _moe_permute_fake(x, sources, positions):
    return x.new_empty((sources.shape[0], x.shape[1]))


@torch.library.custom_op("thingy_b200::moe_combine", mutates_args=())
def moe_combine_op(rows: torch.Tensor, weights: torch.Tensor, sources: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    return moe_combine(rows, weights, MoePlan(sources, positions, None, None, 1))


@moe_combine_op.register_fake
def _moe_combine_fake(rows, weights, sources, positions):
    return rows.new_empty((positions.shape[0], rows.shape[1]))


@torch.library.custom_op("thingy_b200::fp8_grouped_gemm", mutates_args=())
def fp8_grouped_gemm_op(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
                        offsets: torch.Tensor, counts: torch.Tensor, fp32_out: bool) -> torch.Tensor:
    return fp8_grouped_gemm(a, a_scale, b, b_scale, MoePlan(None, None, offsets, counts, 128),
                            out_dtype=torch.float32 if fp32_out else torch.bfloat16)


@fp8_grouped_gemm_op.register_fake
def _fp8_grouped_gemm_fake(a, a_scale, b, b_scale, offsets, counts, fp32_out):
    return a.new_empty((a.shape[0], b.shape[1]), dtype=torch.float32 if fp32_out else torch.bfloat16)


def _reference_op_defined() -> bool:
    try:
        torch.ops.cutie.per_token_fp8_quant
    except (AttributeError, RuntimeError):
        return False
    return True


REFERENCE_NAMESPACE_OP = False
if not _reference_op_defined():

    @torch.library.custom_op("cutie::per_token_fp8_quant", mutates_args=())
    def cutie_per_token_fp8_quant(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        return per_token_cast_to_fp8(x, use_ue8m0=False)

    @cutie_per_token_fp8_quant.register_fake
    def _cutie_per_token_fp8_quant_fake(x):
        return _quantize_fp8_fake(x)

    REFERENCE_NAMESPACE_OP = True
