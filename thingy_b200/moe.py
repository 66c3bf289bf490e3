"""A whole mixture-of-experts layer for few tokens, over 8-bit experts, in one kernel.

``moe_fp8`` takes what ``rms_norm_fp8`` returns for the tokens of a decoding
step (the normalized rows for the router, their codes and scales for the
experts) and the experts' weights in 128 x 128 blocks. No counterpart in the
reference, which stops at the quantizer (src/cutie/rms_norm/bench.py:4-7).
"""

from __future__ import annotations

import torch

from . import _lib
from .fp8_utils import per_block_cast_to_fp8
from .ops import require_binding

MAX_TOKENS = 64
_SCORING = {"softmax": _lib.SCORE_SOFTMAX, "sigmoid": _lib.SCORE_SIGMOID}
_workspaces: dict[tuple[int, int], torch.Tensor] = {}


def moe_workspace(T: int, E: int, top_k: int, H: int, I: int, device=None) -> torch.Tensor:
    """A workspace for ``moe_fp8`` calls of at most these sizes, on the current stream.

    Calls that share one must not overlap on the GPU."""
    device = torch.device("cuda" if device is None else device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    n = require_binding().moe_workspace_bytes(int(T), int(E), int(top_k), int(H), int(I), device.index)
    w = torch.empty(n, dtype=torch.uint8, device=device)
    w[:256].zero_()  # the barrier's count; every call leaves it ready for the next
    return w


def _own_workspace(x, E, top_k, H, I):
    """The current stream's workspace: calls of one stream do not overlap. A captured
    graph gets one of its own, which lives in the graph's memory."""
    sizes = (x.shape[0], E, top_k, H, I)
    with torch.cuda.device(x.device):
        if torch.cuda.is_current_stream_capturing():
            return moe_workspace(*sizes, x.device)
    key = (x.device.index, torch.cuda.current_stream(x.device).cuda_stream)
    w = _workspaces.get(key)
    if w is None or w.numel() < require_binding().moe_workspace_bytes(*sizes, x.device.index):
        w = _workspaces[key] = moe_workspace(*sizes, x.device)
    return w


def clear_moe_workspaces() -> None:
    """Drop the workspaces that ``moe_fp8`` keeps, one a stream, for calls that were given none.

    Each is a block of its stream's, so calls still running on the stream are safe. Also to be
    called before a stream made outside torch is destroyed: another could get its handle.
    """
    _workspaces.clear()


def moe_fp8(
    x: torch.Tensor,
    q: torch.Tensor,
    scale: torch.Tensor,
    router: torch.Tensor,
    w13: torch.Tensor,
    w13_scale: torch.Tensor,
    w2: torch.Tensor,
    w2_scale: torch.Tensor,
    *,
    top_k: int,
    scoring: str = "softmax",
    renormalize: bool = True,
    routed_scale: float = 1.0,
    bias: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    topk_ids: torch.Tensor | None = None,
    topk_weights: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """bf16 [T, H]: router, top-k, the experts' gated MLPs and their weighted sum, T <= 64, on the current stream.

    Forward only: the result carries no gradient, also of an x or router that
    requires one.

    x: bf16 [T, H], the router's input; q, scale: x in e4m3 with 1 x 128 fp32
    scales, any layout (``rms_norm_fp8(..., return_normalized=True)`` gives all
    three). router: bf16 [E, H]; w13: e4m3 [E, 2 I, H] (an expert's gate rows,
    then its up rows); w2: e4m3 [E, H, I]; their scales: fp32 of 128 x 128
    blocks (``quantize_experts``). H and I are multiples of 128, E <= 512,
    top_k <= 16.

    Each token takes the top_k experts of the largest logits, ties to the
    lowest index; ``bias`` (fp32 [E]) is added to the scores for that choice
    only. Its weights are the scores (softmax over all experts, or sigmoid),
    divided by their sum if ``renormalize``, times ``routed_scale``. A NaN
    logit is chosen last; under softmax all weights of its token are NaN. The
    hidden rows silu(gate) * up are cast to e4m3 in 1 x 128 groups; sums are
    fp32, rounded once to bf16. topk_ids (int32) and topk_weights (float32),
    [T, top_k], receive the choices. workspace: ``moe_workspace(...)``;
    without it the call uses one kept for the stream (a fresh one under graph
    capture; ``clear_moe_workspaces`` drops them).
    """
    if scoring not in _SCORING:
        raise ValueError(f"scoring must be one of {tuple(_SCORING)}, got {scoring!r}")
    mod = require_binding()
    if workspace is None:
        if x.dim() != 2 or router.dim() != 2 or w2.dim() != 3 or not x.is_cuda:
            raise ValueError("x and router must be 2-D and w2 3-D CUDA tensors")
        workspace = _own_workspace(x, router.shape[0], int(top_k), x.shape[1], w2.shape[2])
    return mod.moe_fp8(x, q, scale, router, bias, w13, w13_scale, w2, w2_scale, int(top_k),
                       _SCORING[scoring], bool(renormalize), float(routed_scale), out, topk_ids,
                       topk_weights, workspace)


def quantize_experts(w: torch.Tensor, use_ue8m0: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 [E, R, C] -> e4m3 codes [E, R, C] and fp32 scales [E, R/128, C/128] of 128 x 128 blocks."""
    if w.dim() != 3 or w.shape[1] % 128 != 0 or w.shape[2] % 128 != 0:
        raise ValueError(f"w must be [E, R, C] with R and C multiples of 128, got {tuple(w.shape)}")
    E, R, C = w.shape
    q, s = per_block_cast_to_fp8(w.reshape(E * R, C), use_ue8m0)
    return q.view(E, R, C), s.view(E, R // 128, C // 128)
