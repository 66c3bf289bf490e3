"""The workspaces that moe_fp8 keeps for streams, and how to be rid of them."""

import pytest
import torch

import thingy_b200 as tb
from thingy_b200.moe import quantize_experts

pytestmark = pytest.mark.gpu


def _layer(T=16, E=8, H=512, I=256):
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    q, s, _, n = tb.rms_norm_fp8(x, torch.ones(H, dtype=torch.bfloat16, device="cuda"), 1e-6, return_normalized=True)
    router = torch.randn(E, H, generator=g, device="cuda").to(torch.bfloat16)
    w13 = quantize_experts((0.05 * torch.randn(E, 2 * I, H, generator=g, device="cuda")).to(torch.bfloat16))
    w2 = quantize_experts((0.05 * torch.randn(E, H, I, generator=g, device="cuda")).to(torch.bfloat16))
    return n, q, s, router, *w13, *w2


def test_kept_workspaces_can_be_dropped():
    ops = _layer()
    tb.clear_moe_workspaces()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    want = tb.moe_fp8(*ops, top_k=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = tb.moe_fp8(*ops, top_k=2)
    torch.cuda.current_stream().wait_stream(side)
    results = 2 * want.numel() * want.element_size()
    kept = torch.cuda.memory_allocated() - before - results
    assert kept >= 2 * 16 * 2 * 512 * 4  # the down products of two streams at the least
    tb.clear_moe_workspaces()  # the side stream's call may still run: its block stays that stream's
    assert torch.cuda.memory_allocated() - before == results
    assert torch.equal(tb.moe_fp8(*ops, top_k=2), want) and torch.equal(other, want)
    torch.cuda.synchronize()
    tb.clear_moe_workspaces()


def test_result_carries_no_gradient():
    ops = list(_layer())
    want = tb.moe_fp8(*ops, top_k=2)
    ops[0] = ops[0].clone().requires_grad_()
    ops[3] = ops[3].clone().requires_grad_()
    y = tb.moe_fp8(*ops, top_k=2)
    assert not y.requires_grad and torch.equal(y, want)
