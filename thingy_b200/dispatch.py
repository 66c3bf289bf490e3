"""Tokens sorted by expert and back: what lies between a router and experts with many tokens.

``moe_sort`` turns the router's choices into a plan, ``moe_permute`` brings the
tokens' rows into the experts' order and ``moe_combine`` brings the experts'
results back, weighted and summed; both are differentiable. The products in
between are ``fp8_grouped_linear`` (training) and ``fp8_grouped_gemm`` (codes).
For a decode step of at most 64 tokens ``moe_fp8`` is the whole layer in one
kernel. No counterpart in the reference, which stops at the quantizer
(src/cutie/rms_norm/bench.py:4-7).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .ops import require_binding


class MoePlan(NamedTuple):
    """Where sorted rows come from and go to; int32 tensors on the GPU.

    sources [R]: the choice t * k + j that a sorted row holds, -1 in padding.
    positions [T, k]: the sorted row of each choice, -1 where it is absent.
    offsets [E + 1]: where each expert's rows begin, multiples of ``align``.
    counts [E]: how many rows each expert has, without its padding.

    ``moe_sort`` makes one. A program may make its own, for a fixed capacity an
    expert, say: offsets that do not decrease, sources and positions that name each
    other, rows of an expert from its offset on and padding behind them.
    """

    sources: torch.Tensor
    positions: torch.Tensor
    offsets: torch.Tensor
    counts: torch.Tensor
    align: int


def moe_plan_rows(T: int, top_k: int, num_experts: int, align: int = 1) -> int:
    """R of a plan: the most sorted rows that any choices of these sizes need."""
    return require_binding().moe_plan_rows(int(T), int(top_k), int(num_experts), int(align))


def moe_sort(topk_ids: torch.Tensor, num_experts: int, *, align: int = 1) -> MoePlan:
    """The plan that sorts the choices by expert, on the current stream and without a copy to the host.

    topk_ids: int32 or int64 [T, k], any number of choices of the same expert;
    an id outside [0, num_experts) is an absent choice (dropped, or another
    rank's). Choices of one expert keep their order t * k + j. Every expert's
    rows begin at a multiple of ``align`` (``fp8_grouped_linear`` and
    ``fp8_grouped_gemm`` take 128). R = ``moe_plan_rows(T, k, num_experts,
    align)`` rows, whatever the ids; rows that hold no choice are padding.
    num_experts <= 512.
    """
    return MoePlan(*require_binding().moe_sort(topk_ids, int(num_experts), int(align), False), int(align))


def moe_permute(x: torch.Tensor, plan: MoePlan) -> torch.Tensor:
    """[R, H]: row r is x's row of the token whose choice sorted row r holds; zeros in padding.

    x: [T, H] of 1-, 2- or 4-byte elements (rows of activations; also codes, and
    their scales with a token a row), any strides. Differentiable for bf16, fp16
    and fp32: a token's gradient is the sum of its rows', in fp32 in the order
    of j, rounded once.
    """
    return require_binding().moe_permute(x, plan.sources, plan.positions)


def moe_combine(rows: torch.Tensor, weights: torch.Tensor, plan: MoePlan) -> torch.Tensor:
    """[T, H]: token t's sum over j of weights[t, j] * rows[positions[t, j]], absent choices left out.

    rows: bf16, fp16 or fp32 [R, H], any strides; weights: float32 [T, k]. The sum
    runs in fp32 in the order of j and is rounded once. Differentiable in rows
    (zeros in padding) and weights (fp32 dot products; 0 for absent choices).
    """
    return require_binding().moe_combine(rows, weights, plan.sources, plan.positions)
