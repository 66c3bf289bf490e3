"""cutie_set_wait_limit reaches the block-scaled product and the experts' kernel.

With a limit of -1 every wait that would have to block gives up at once: the launch records device
error 1, lets its own copies land and returns. The same call with the default limit, on the same
workspace, then gives the earlier bits.
"""

import pytest
import torch

import thingy_b200 as tb
from thingy_b200 import _lib
from thingy_b200.moe import quantize_experts

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def _runs_out_then_clean(call):
    want = call()
    torch.cuda.synchronize()
    assert _lib.device_error(clear=True) == 0
    prev = _lib.set_wait_limit(-1)
    try:
        call()
    finally:
        _lib.set_wait_limit(prev)
    torch.cuda.synchronize()
    assert _lib.device_error(clear=True) == 1, "no wait ran out"
    for _ in range(2):
        got = call()
        torch.cuda.synchronize()
        assert _lib.device_error(clear=True) == 0
        assert torch.equal(got, want)


def _operands(M, N, K, kind):
    g = torch.Generator(device="cuda").manual_seed(M + N + K)

    def codes(rows):
        return (60.0 * torch.randn(rows, K, generator=g, device="cuda")).clamp(-448, 448).to(F8)

    def scales(rows):
        return 0.01 * (0.1 + torch.rand(rows, -(-K // 128), generator=g, device="cuda"))

    return codes(M), scales(M), codes(N), scales(N if kind == "rows" else -(-N // 128))


@pytest.mark.parametrize("what,M,N,K,kind", [
    ("few rows, K split", 8, 5120, 5120, "blocks"),
    ("few rows, one rank", 24, 32768, 512, "blocks"),
    ("few rows, 64 columns", 64, 2048, 4096, "blocks"),
    ("128-wide tiles", 1000, 1152, 384, "blocks"),
    ("128-wide tiles, a scale a row", 1000, 1150, 400, "rows"),
    ("128-wide tiles, K split", 200, 300, 7168, "blocks"),
    ("128-wide tiles, K split, a scale a row", 513, 130, 8192, "rows"),
    ("256-wide tiles by pairs", 2560, 2560, 1024, "blocks"),
    ("256-wide tiles by pairs, odd columns, a scale a row", 2560, 2561, 1024, "rows"),
    ("256-wide tiles by pairs, then the rest in 128-wide ones", 2300, 2304, 4224, "blocks"),
])
def test_product_wait_runs_out_then_clean_launch(what, M, N, K, kind):
    ops = _operands(M, N, K, kind)
    _runs_out_then_clean(lambda: tb.fp8_block_gemm(*ops))


@pytest.mark.parametrize("T,E,k,H,I", [(1, 16, 4, 1024, 512), (8, 8, 2, 2048, 256), (9, 8, 2, 1024, 256),
                                       (24, 12, 3, 896, 384), (64, 16, 4, 1024, 256)])
def test_experts_wait_runs_out_then_clean_launch(T, E, k, H, I):
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    q, s, _, n = tb.rms_norm_fp8(x, torch.ones(H, dtype=torch.bfloat16, device="cuda"), 1e-6, return_normalized=True)
    router = (0.05 * torch.randn(E, H, generator=g, device="cuda")).to(torch.bfloat16)
    w13 = quantize_experts((0.05 * torch.randn(E, 2 * I, H, generator=g, device="cuda")).to(torch.bfloat16))
    w2 = quantize_experts((0.05 * torch.randn(E, H, I, generator=g, device="cuda")).to(torch.bfloat16))
    workspace = tb.moe_workspace(T, E, k, H, I)
    _runs_out_then_clean(lambda: tb.moe_fp8(n, q, s, router, *w13, *w2, top_k=k, workspace=workspace))
