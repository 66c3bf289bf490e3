"""fp8_grouped_linear on plans whose experts begin at multiples of 256 and more.

An expert may then have whole tiles of 128 rows that are padding; they count as zeros, in the
weight gradient too. The memory that the casts write into holds NaN before.
"""

import pytest
import torch

import thingy_b200 as tb
from test_grouped_gemm_gpu import check, quantized

pytestmark = pytest.mark.gpu


def fill_free_memory_with_nan():
    """What the allocator gives out next holds bytes of 255: NaN as e4m3, bf16 and fp32."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    blocks = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in [1 << 19] * 64 + [1 << 23] * 16 + [1 << 27] * 4]
    torch.cuda.synchronize()
    del blocks


def ids_of(counts, extra=33):
    ids = torch.cat([torch.full((c,), e, dtype=torch.int32) for e, c in enumerate(counts)] +
                    [torch.full((extra,), -1, dtype=torch.int32)])
    return ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(len(ids)))].reshape(-1, 1).cuda()


@pytest.mark.parametrize("weight_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,K", [(128, 128), (384, 256), (2048, 2048)])
@pytest.mark.parametrize("align", [256, 384, 1024])
@pytest.mark.parametrize("counts", [[100], [1, 0, 257, 128, 129], [7] * 20, [600, 0, 0, 3]])
def test_linear_and_gradients(counts, align, N, K, weight_dtype):
    E, ids = len(counts), ids_of(counts)
    g = torch.Generator(device="cuda").manual_seed(N + K)
    tokens = torch.randn(len(ids), K, generator=g, device="cuda").bfloat16()
    grads = (0.1 * torch.randn(len(ids), N, generator=g, device="cuda")).bfloat16()
    w = (0.02 * torch.randn(E, N, K, generator=g, device="cuda")).to(weight_dtype).requires_grad_()
    dws = {}
    for a in (128, align):
        plan = tb.moe_sort(ids, E, align=a)
        pad = plan.sources < 0
        x, dy = tb.moe_permute(tokens, plan), tb.moe_permute(grads, plan)
        x[pad], dy[pad] = float("nan"), float("inf")
        x.requires_grad_()
        fill_free_memory_with_nan()
        y = tb.fp8_grouped_linear(x, w, plan)
        dx, dws[a] = torch.autograd.grad(y, (x, w), dy)
        x0, dy0 = x.detach().masked_fill(pad[:, None], 0), dy.masked_fill(pad[:, None], 0)
        off = plan.offsets.tolist()
        for e in range(E):
            rows = slice(off[e], off[e + 1])
            if not counts[e]:
                assert bool((dws[a][e] == 0).all())
                continue
            we = quantized(w[e].detach().bfloat16(), 128, 128)
            check(y[rows].detach(), quantized(x0[rows], 1, 128), we, torch.bfloat16)
            check(dx[rows], quantized(dy0[rows], 1, 128, True), we.t(), torch.bfloat16)
            check(dws[a][e], quantized(dy0[rows], 128, 1, True).t(), quantized(x0[rows], 128, 1).t(), weight_dtype)
        assert bool((y[pad] == 0).all()) and bool((dx[pad] == 0).all())
    # the tiles of the weight gradient do not depend on the rows, and whole tiles of padding add zeros
    assert torch.equal(dws[128], dws[align])


def test_every_tile_of_the_sorted_cast_is_written():
    """Codes of padding are zeros wherever it lies: within an expert, between experts, behind the last."""
    lib, R, H = tb._lib.load(), 1024, 256
    sources = torch.full((R,), -1, dtype=torch.int32, device="cuda")
    for first, n in ((0, 100), (384, 3), (640, 1)):
        sources[first : first + n] = torch.arange(n, dtype=torch.int32, device="cuda")
    x = torch.randn(R, H, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").bfloat16()
    x[sources < 0] = float("nan")
    for fmt, least in ((tb._lib.SCALE_FP32, 1e-4), (tb._lib.SCALE_FP32 + tb._lib.SCALE_GRADIENT, 2.0**-92)):
        q, qt = (torch.full(s, 255, dtype=torch.uint8, device="cuda") for s in ((R, H), (H, R)))
        s, st = (torch.full(t, float("nan"), device="cuda") for t in ((H // 128, R), (R // 128, H)))
        tb._lib.check(lib.cutie_cast_fp8_sorted(x.data_ptr(), H, R, H, sources.data_ptr(), fmt, q.data_ptr(), H, s.data_ptr(), R,
                                                qt.data_ptr(), R, st.data_ptr(), H, torch.cuda.current_stream().cuda_stream))
        pad = sources < 0
        assert bool((q[pad] == 0).all()) and bool((qt[:, pad] == 0).all())
        assert bool((s[:, pad] == torch.tensor(least, device="cuda")).all())
        assert not bool(torch.isnan(s).any()) and not bool(torch.isnan(st).any())
        empty = [i for i in range(R // 128) if bool(pad[128 * i : 128 * i + 128].all())]
        assert empty == [1, 2, 4, 6, 7] and bool((st[empty] == torch.tensor(least, device="cuda")).all())
