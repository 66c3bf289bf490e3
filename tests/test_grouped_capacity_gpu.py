"""The experts' products on plans of a fixed capacity an expert, some of them empty, made without moe_sort.

Padding is zero from both kernels (few rows an expert, and tiles), and so are rows before the first expert's."""

import pytest
import torch

import thingy_b200 as tb
from test_grouped_align_gpu import fill_free_memory_with_nan
from test_grouped_gemm_gpu import check, codes, dequant_blocks, dequant_rows, quantized

pytestmark = pytest.mark.gpu


def capacity_plan(counts, capacity, before=0, behind=0):
    """Expert e's rows begin at before + e * capacity; `behind` rows follow the last."""
    E = len(counts)
    sources = torch.full((before + E * capacity + behind,), -1, dtype=torch.int32)
    positions, at = torch.zeros(sum(counts), 1, dtype=torch.int32), 0
    for e, n in enumerate(counts):
        first = before + e * capacity
        sources[first : first + n] = torch.arange(at, at + n, dtype=torch.int32)
        positions[at : at + n, 0] = torch.arange(first, first + n, dtype=torch.int32)
        at += n
    offsets = before + capacity * torch.arange(E + 1, dtype=torch.int32)
    return tb.MoePlan(sources.cuda(), positions.cuda(), offsets.int().cuda(), torch.tensor(counts, dtype=torch.int32).cuda(), 128)


# capacities of 128 go to the kernel for few rows an expert, larger ones to the tiles
PLANS = [([0, 5, 0, 128, 1, 0], 128, 0, 0), ([0], 128, 0, 0), ([0, 5, 0, 200, 1, 0], 256, 0, 0), ([3, 0, 0], 128, 128, 128),
         ([0, 300, 0, 1], 384, 256, 128), ([1] + [0] * 99, 128, 0, 0), ([0] * 40 + [90], 128, 384, 0)]


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,K", [(16, 128), (304, 528), (1024, 512)])
@pytest.mark.parametrize("counts,capacity,before,behind", PLANS)
def test_product(counts, capacity, before, behind, N, K, out_dtype):
    E, plan = len(counts), capacity_plan(counts, capacity, before, behind)
    R, KB = plan.sources.shape[0], -(-K // 128)
    g = torch.Generator(device="cuda").manual_seed(N + K)
    a, sa = codes(g, R, K), torch.rand(R, KB, generator=g, device="cuda") + 0.5
    a[plan.sources < 0] = torch.tensor(float("nan")).to(a.dtype).cuda()
    b, sb = codes(g, E, N, K), torch.rand(E, -(-N // 128), KB, generator=g, device="cuda") + 0.5
    wide = torch.full((R + 2, N), float("nan"), dtype=out_dtype, device="cuda")
    out = wide[1:-1]
    tb.fp8_grouped_gemm(a, sa, b, sb, plan, out=out)
    for e, n in enumerate(counts):
        rows = slice(before + e * capacity, before + e * capacity + n)
        if n:
            check(out[rows], dequant_rows(a[rows], sa[rows]), dequant_blocks(b[e], sb[e]), out_dtype)
    assert bool((out[plan.sources < 0] == 0).all())
    assert bool(wide[0].isnan().all()) and bool(wide[-1].isnan().all())


@pytest.mark.parametrize("counts,capacity,before,behind", PLANS)
def test_linear_and_gradients(counts, capacity, before, behind):
    E, N, K, plan = len(counts), 256, 384, capacity_plan(counts, capacity, before, behind)
    R, pad = plan.sources.shape[0], plan.sources < 0
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(R, K, generator=g, device="cuda").bfloat16()
    dy = (0.1 * torch.randn(R, N, generator=g, device="cuda")).bfloat16()
    x[pad], dy[pad] = float("nan"), float("inf")
    x.requires_grad_()
    w = (0.02 * torch.randn(E, N, K, generator=g, device="cuda")).requires_grad_()
    fill_free_memory_with_nan()
    y = tb.fp8_grouped_linear(x, w, plan)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert bool((y[pad] == 0).all()) and bool((dx[pad] == 0).all())
    x0, dy0 = x.detach().masked_fill(pad[:, None], 0), dy.masked_fill(pad[:, None], 0)
    for e, n in enumerate(counts):
        rows = slice(before + e * capacity, before + (e + 1) * capacity)
        if not n:
            assert bool((dw[e] == 0).all())
            continue
        we = quantized(w[e].detach().bfloat16(), 128, 128)
        check(y[rows].detach(), quantized(x0[rows], 1, 128), we, torch.bfloat16)
        check(dx[rows], quantized(dy0[rows], 1, 128, True), we.t(), torch.bfloat16)
        check(dw[e], quantized(dy0[rows], 128, 1, True).t(), quantized(x0[rows], 128, 1).t(), torch.float32)
