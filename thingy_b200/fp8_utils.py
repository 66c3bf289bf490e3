"""Drop-in for the activation quantizer of src/cutie/vendor/prime_rl/fp8_utils.py.

``per_token_cast_to_fp8(x, use_ue8m0, gran_k=128)`` returns the same
``(out e4m3 [M, H], sf fp32 [M, ceil(H/gran_k)])`` as
``per_token_cast_to_fp8_triton`` (fp8_utils.py:63-89): per (row, gran_k
group) amax, ``s = max(amax/448, 1e-4)``, ``2^ceil(log2 s)`` when use_ue8m0,
``e4m3(x / s)``; a partial last group is reduced over its valid columns only.
It runs the hand-written sm_100a kernel; gran_k may also be 32 or 64.

``per_block_cast_to_fp8`` (weights, 128 x 128 blocks) and ``two_way_cast_to_fp8``
(activations and gradients, 1 x 128 groups along both axes) make the operands
of ``thingy_b200.fp8_block_gemm`` by the same rule (on request with scales for
small gradients); they have no counterpart in the reference, which quantizes
activations along their rows only.
"""

from __future__ import annotations

import torch

from .fused import empty_scale
from .ops import FP8_DTYPE, launch_rms_norm_fp8, require_binding

GROUP_ALIGNMENT = 128


def ceil_div(x: int, y: int) -> int:
    return (x + y - 1) // y


def per_token_cast_to_fp8(
    x: torch.Tensor, use_ue8m0: bool, gran_k: int = GROUP_ALIGNMENT
) -> tuple[torch.Tensor, torch.Tensor]:
    assert x.dim() == 2
    assert gran_k in (32, 64, 128)
    rows, cols = x.shape
    out = torch.empty_like(x, dtype=FP8_DTYPE)
    sf = empty_scale(rows, cols, gran_k, "ue8m0" if use_ue8m0 else "fp32", "row", x.device)
    launch_rms_norm_fp8(
        x, None, 0.0, q=out, scale=sf, group_size=gran_k,
        scale_format="ue8m0" if use_ue8m0 else "fp32", scale_layout="row", normalize=False,
    )
    return out, sf


# The name the reference's callers import (fp8_utils.py:63).
per_token_cast_to_fp8_triton = per_token_cast_to_fp8


def per_block_cast_to_fp8(w: torch.Tensor, use_ue8m0: bool = False, transposed: bool = False):
    """bf16 [N, K] -> e4m3 codes [N, K] and fp32 scales [ceil(N/128), ceil(K/128)] of 128 x 128 blocks.

    With ``transposed`` returns (q, s, qt, st): also the codes [K, N] of w's
    transpose and their scales [ceil(K/128), ceil(N/128)] (a layer's input
    gradient contracts over N). K must be a multiple of 8; the codes' rows
    start on 16-byte boundaries (a view of a wider buffer when the width is
    not a multiple of 16). Runs on the current stream.
    """
    q, s, qt, st = require_binding().cast_fp8_tiles(w, True, bool(use_ue8m0), bool(transposed), False)
    return (q, s, qt, st) if transposed else (q, s)


def two_way_cast_to_fp8(x: torch.Tensor, use_ue8m0: bool = False, gradient: bool = False):
    """bf16 [M, H] -> (q, s, qt, st): e4m3 codes in 1 x 128 groups along the rows and along the columns.

    q [M, H] with s [M, ceil(H/128)] quantizes rows (the forward product and
    the input gradient contract over H); qt [H, M] with st [H, ceil(M/128)]
    the rows of x's transpose (the weight gradient contracts over M). x is
    read once. Scales are group-major views (strides (1, M) and (1, H)), the
    codes' rows start on 16-byte boundaries. H must be a multiple of 8. With
    ``gradient`` a group whose maximum is below 1e-4 has the scale max(amax/448,
    2^-92) instead of 1e-4, at which values below 9.8e-8 become zero. Runs on
    the current stream.
    """
    return require_binding().cast_fp8_tiles(x, False, bool(use_ue8m0), True, bool(gradient))
