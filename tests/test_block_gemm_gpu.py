"""The block-scaled FP8 product, the casts that make its operands and the linear
layer over them, against plain forms in 64 bits.

Tolerances. Products: the inner sum of a 128-wide block is fp32 in any order
(at most 128 roundings of the partial sums, each bounded by the block's sum of
magnitudes), the outer sum one fp32 rounding a block, then the rounding to the
output type: |err| <= |ref| 2^-8 (bf16, half an ulp is 2^-9) or 2^-23 (fp32)
plus mag (128 + KB) 2^-23, mag the sum of the terms' magnitudes. Casts: bit
for bit against the rule evaluated on the CPU in fp32 (correctly rounded
division there).
"""

import pytest
import torch

import thingy_b200 as tb

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def _cast_ref(x, rows, cols, pow2):
    """Codes and scales of rows x cols tiles on the CPU: fp32 division, round to nearest even."""
    x = x.float().cpu()
    R, C = x.shape
    full = torch.zeros(-(-R // rows) * rows, -(-C // cols) * cols)
    full[:R, :C] = x
    amax = full.view(full.shape[0] // rows, rows, full.shape[1] // cols, cols).abs()
    amax = amax.permute(0, 2, 1, 3).flatten(2).amax(2)
    s = torch.clamp_min(amax / 448.0, 1e-4)
    if pow2:
        m, e = torch.frexp(s)
        s = torch.ldexp(torch.ones_like(s), torch.where(m == 0.5, e - 1, e))
    spread = s[:, None, :, None].expand(-1, rows, -1, cols).reshape(full.shape)[:R, :C]
    return (x / spread).to(F8), s


def _same(got, want):
    assert tuple(got.shape) == tuple(want.shape)
    assert torch.equal(got.cpu().contiguous().view(torch.uint8), want.contiguous().view(torch.uint8))


def _matrix(M, H, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, H, generator=g) * scale
    if H > 100:
        x[:, torch.randperm(H, generator=g)[: H // 100]] *= 50.0
    return x.to(torch.bfloat16)


SHAPES = [(1, 8), (1, 128), (7, 136), (127, 1032), (128, 128), (129, 256), (300, 2056), (1000, 640)]


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("M,H", SHAPES)
def test_two_way_cast(M, H, pow2):
    x = _matrix(M, H, seed=M + H)
    q, s, qt, st = tb.two_way_cast_to_fp8(x.cuda(), pow2)
    wq, ws = _cast_ref(x, 1, 128, pow2)
    _same(q, wq)
    assert torch.equal(s.cpu(), ws)
    wq, ws = _cast_ref(x.t(), 1, 128, pow2)
    _same(qt, wq)
    assert torch.equal(st.cpu(), ws)


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("M,H", SHAPES)
def test_block_cast(M, H, pow2):
    x = _matrix(M, H, seed=M * H, scale=0.02)
    wq, ws = _cast_ref(x, 128, 128, pow2)
    q, s = tb.per_block_cast_to_fp8(x.cuda(), pow2)
    _same(q, wq)
    assert torch.equal(s.cpu(), ws)
    q, s, qt, st = tb.per_block_cast_to_fp8(x.cuda(), pow2, transposed=True)
    _same(q, wq)
    _same(qt, wq.t())
    assert torch.equal(s.cpu(), ws) and torch.equal(st.cpu(), ws.t())


def test_casts_agree_with_the_row_quantizer():
    x = _matrix(333, 1024, seed=4).cuda()
    q0, s0 = tb.per_token_cast_to_fp8(x, False)
    q, s, _, _ = tb.two_way_cast_to_fp8(x)
    _same(q, q0.cpu())
    assert torch.equal(s, s0)


def test_casts_of_strided_rows_zeros_and_tiny_values():
    wide = _matrix(200, 512, seed=9).cuda()
    x = wide[:, 64:320]
    x[3] = 0.0
    x[:, 5] = 0.0
    x[7] = 1e-30
    q, s, qt, st = tb.two_way_cast_to_fp8(x)
    wq, ws = _cast_ref(x.cpu(), 1, 128, False)
    _same(q, wq)
    assert torch.equal(s.cpu(), ws)
    wq, ws = _cast_ref(x.cpu().t(), 1, 128, False)
    _same(qt, wq)
    assert torch.equal(st.cpu(), ws)


def test_casts_of_nonfinite_values():
    x = _matrix(130, 256, seed=2)
    x[1, 3] = float("nan")
    x[5, 200] = float("inf")
    q, s, qt, st = tb.two_way_cast_to_fp8(x.cuda())
    q, s, qt, st = q.float().cpu(), s.cpu(), qt.float().cpu(), st.cpu()
    assert torch.isnan(q[1, 3]) and torch.isnan(qt[3, 1])
    assert torch.isinf(s[5, 1]) and torch.isinf(st[200, 0])
    assert torch.isnan(q[5, 128:]).all() and torch.isnan(qt[200, :128]).all()
    # every other group is as without them
    clean = x.clone()
    clean[1, 3] = 0.0
    wq, ws = _cast_ref(clean, 1, 128, False)
    rest = torch.ones(130, 256, dtype=torch.bool)
    rest[1, 3] = False
    rest[5, 128:] = False
    assert torch.equal(q[rest], wq.float()[rest])
    keep = torch.ones(130, 2, dtype=torch.bool)
    keep[5, 1] = False
    assert torch.equal(s[keep], ws[keep])


def test_empty_casts():
    x = torch.empty(0, 256, dtype=torch.bfloat16, device="cuda")
    q, s, qt, st = tb.two_way_cast_to_fp8(x)
    assert q.shape == (0, 256) and s.shape == (0, 2) and qt.shape == (256, 0) and st.shape == (256, 0)
    q, s, qt, st = tb.per_block_cast_to_fp8(x, transposed=True)
    assert q.shape == (0, 256) and s.shape == (0, 2) and qt.shape == (256, 0) and st.shape == (2, 0)


def test_cast_refusals():
    x = torch.zeros(4, 128, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="multiple of 8"):
        tb.two_way_cast_to_fp8(torch.zeros(4, 132, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError, match="bfloat16"):
        tb.two_way_cast_to_fp8(x.float())
    with pytest.raises(ValueError, match="2-D"):
        tb.per_block_cast_to_fp8(x[0])
    with pytest.raises(ValueError, match="contiguous along"):
        tb.per_block_cast_to_fp8(x.t())
    with pytest.raises(ValueError, match="overlapping"):
        tb.two_way_cast_to_fp8(x[:1].expand(4, 128))
    with pytest.raises(ValueError, match="CUDA"):
        tb.two_way_cast_to_fp8(x.cpu())
    with pytest.raises(ValueError, match="aligned"):
        tb.two_way_cast_to_fp8(torch.zeros(4, 136, dtype=torch.bfloat16, device="cuda")[:, 4:132])


# ------------------------------------------------------------------ products


def _padded(q):
    """Rows on 16-byte boundaries."""
    out = torch.zeros(q.shape[0], -(-q.shape[1] // 16) * 16, dtype=q.dtype, device=q.device)
    out[:, : q.shape[1]] = q
    return out[:, : q.shape[1]]


def _operands(M, N, K, kind, seed, layout="row"):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def codes(rows):
        return _padded((60.0 * torch.randn(rows, K, generator=g, device="cuda")).clamp(-448, 448).to(F8))

    KB = -(-K // 128)

    def scales(rows):
        s = 0.01 * (0.1 + torch.rand(rows, KB, generator=g, device="cuda"))
        return s.t().contiguous().t() if layout == "col" else s

    return codes(M), scales(M), codes(N), scales(N if kind == "rows" else -(-N // 128))


def _reference(a, sa, b, sb):
    K, N = a.shape[1], b.shape[0]
    A = a.double() * sa.double().repeat_interleave(128, 1)[:, :K]
    rows = sb if sb.shape[0] == N else sb.repeat_interleave(128, 0)[:N]
    B = b.double() * rows.double().repeat_interleave(128, 1)[:, :K]
    return A @ B.t(), A.abs() @ B.abs().t()


def _check(d, a, sa, b, sb, base=None):
    ref, mag = _reference(a, sa, b, sb)
    if base is not None:
        ref = ref + base.double()
        mag = mag + base.double().abs()
    K = a.shape[1]
    rel = 2.0**-8 if d.dtype == torch.bfloat16 else 2.0**-22
    bound = ref.abs() * rel + mag * ((128 + -(-K // 128)) * 2.0**-23) + 1e-30
    err = (d.double() - ref).abs()
    assert bool((err <= bound).all()), f"max excess {(err - bound).max().item():.3e}"


PRODUCTS = [
    (1, 128, 128), (1, 5120, 5120), (3, 8, 16), (5, 1000, 384), (8, 136, 2048), (16, 256, 7168),
    (17, 257, 1040), (24, 640, 640), (32, 384, 129), (33, 129, 1000), (48, 2048, 4096),
    (64, 5120, 5120), (65, 130, 160), (100, 1024, 2048), (128, 128, 7168), (129, 100, 48),
    (200, 1000, 1000), (1000, 384, 7168),
    # few tiles and a long K: K split over a cluster, ragged tiles, uneven K ranges
    (128, 2048, 7168), (2500, 2304, 4100), (6500, 800, 4112), (150, 333, 2900), (513, 130, 2561), (300, 1000, 4096), (257, 385, 16400), (2049, 2100, 272), (4800, 8192, 512), (4097, 9000, 400),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_block_product(M, N, K, dtype):
    ops = _operands(M, N, K, "blocks", seed=M + N + K, layout="col" if M % 2 else "row")
    _check(tb.fp8_block_gemm(*ops, out_dtype=dtype), *ops)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(2, 3, 5), (128, 128, 128), (129, 100, 48), (130, 515, 1001),
                                   (640, 300, 2056), (2049, 2100, 272), (4097, 9000, 400),
                                   (512, 512, 8200), (131, 77, 5001), (640, 515, 2600),
                                   (2500, 2303, 4100)])
def test_group_product(M, N, K, dtype):
    ops = _operands(M, N, K, "rows", seed=M * 3 + N + K, layout="col" if N % 2 else "row")
    _check(tb.fp8_block_gemm(*ops, out_dtype=dtype), *ops)


@pytest.mark.parametrize("M,N,K,kind", [(9, 300, 640, "blocks"), (700, 515, 1000, "rows"),
                                        (300, 264, 512, "blocks"), (200, 264, 4096, "blocks"),
                                        (200, 263, 4100, "rows")])
def test_accumulation(M, N, K, kind):
    ops = _operands(M, N, K, kind, seed=K)
    base = torch.randn(M, N, device="cuda")
    out = base.clone()
    got = tb.fp8_block_gemm(*ops, out=out, accumulate=True)
    assert got is out or got.data_ptr() == out.data_ptr()
    _check(out, *ops, base=base)


@pytest.mark.parametrize("M,K", [(3, 256), (200, 256), (200, 4096)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_output_is_written_between_its_columns_only(M, K, dtype):
    ops = _operands(M, 200, K, "blocks", seed=7)
    wide = torch.full((M, 209), -7.0, dtype=dtype, device="cuda")
    tb.fp8_block_gemm(*ops, out=wide[:, 3:203])
    _check(wide[:, 3:203], *ops)
    assert bool((wide[:, :3] == -7).all()) and bool((wide[:, 203:] == -7).all())


def test_strided_operands():
    a, sa, b, sb = _operands(150, 260, 512, "blocks", seed=8)
    wa = torch.zeros(150, 1024, dtype=F8, device="cuda")
    wa[:, 256:768] = a
    d = tb.fp8_block_gemm(wa[:, 256:768], sa, b, sb)
    assert torch.equal(d, tb.fp8_block_gemm(a, sa, b, sb))


def test_empty_products():
    for M, N, K in [(0, 128, 128), (4, 0, 128)]:
        ops = _operands(M, N, K, "blocks", seed=1)
        assert tb.fp8_block_gemm(*ops).shape == (M, N)
    ops = _operands(4, 100, 0, "blocks", seed=1)
    assert bool((tb.fp8_block_gemm(*ops) == 0).all())
    out = torch.ones(4, 100, device="cuda")
    tb.fp8_block_gemm(*ops, out=out, accumulate=True)
    assert bool((out == 1).all())


def test_nan_codes_reach_their_rows_and_columns_only():
    a, sa, b, sb = _operands(5, 300, 256, "blocks", seed=3)
    a[2, 17] = float("nan")
    b[44, 130] = float("nan")
    d = tb.fp8_block_gemm(a, sa, b, sb)
    nan = torch.isnan(d)
    want = torch.zeros_like(nan)
    want[2] = True
    want[:, 44] = True
    assert torch.equal(nan, want)


def test_another_stream_and_graph():
    ops = _operands(16, 512, 1024, "blocks", seed=5)
    want = tb.fp8_block_gemm(*ops)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = tb.fp8_block_gemm(*ops)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tb.fp8_block_gemm(*ops, out=out)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_product_is_the_same_every_time():
    for M, N, K in [(20, 1000, 7168), (900, 700, 4096), (200, 300, 7168)]:
        ops = _operands(M, N, K, "blocks", seed=6)
        first = tb.fp8_block_gemm(*ops)
        for _ in range(5):
            assert torch.equal(tb.fp8_block_gemm(*ops), first)


def test_product_refusals():
    a, sa, b, sb = _operands(8, 256, 256, "blocks", seed=1)
    for args, what in [
        ((a.float(), sa, b, sb), "float8"),
        ((a, sa, b[:, :128], sb), "columns"),
        ((a, sa[:, :1], b, sb), "a_scale"),
        ((a, sa, b, sb[:1]), "b_scale"),
        ((a, sa.half(), b, sb), "float32"),
        ((a.cpu(), sa, b, sb), "CUDA"),
        ((a, sa.cpu(), b, sb), "device"),
        ((a.t(), sa, b, sb), "contiguous"),
        ((a[:1].expand(8, 256), sa, b, sb), "overlapping"),
    ]:
        with pytest.raises(ValueError, match=what):
            tb.fp8_block_gemm(*args)
    odd = torch.zeros(8, 264, dtype=F8, device="cuda")
    with pytest.raises(ValueError, match="aligned"):
        tb.fp8_block_gemm(odd[:, :256], sa, b, sb)
    with pytest.raises(ValueError, match="out_dtype"):
        tb.fp8_block_gemm(a, sa, b, sb, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="accumulat"):
        tb.fp8_block_gemm(a, sa, b, sb, accumulate=True)
    with pytest.raises(ValueError, match="fp32"):
        tb.fp8_block_gemm(a, sa, b, sb, out=torch.zeros(8, 256, dtype=torch.bfloat16, device="cuda"),
                          accumulate=True)
    with pytest.raises(ValueError, match="out must have shape"):
        tb.fp8_block_gemm(a, sa, b, sb, out=torch.zeros(8, 255, device="cuda"))


# ------------------------------------------------------------------ the linear layer


def _dequant(q, s, tile):
    R, C = q.shape
    return q.double() * s.double().repeat_interleave(tile[0], 0)[:R].repeat_interleave(128, 1)[:, :C]


@pytest.mark.parametrize("M,N,K,wdtype", [(1, 128, 128, torch.bfloat16), (77, 264, 136, torch.bfloat16),
                                          (300, 512, 1024, torch.float32), (1001, 776, 520, torch.bfloat16)])
def test_linear_and_its_gradients(M, N, K, wdtype):
    x = _matrix(M, K, seed=1).cuda().requires_grad_()
    w = (_matrix(N, K, seed=2, scale=0.02).cuda()).to(wdtype).requires_grad_()
    dy = _matrix(M, N, seed=3, scale=0.1).cuda()
    y = tb.fp8_linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert y.dtype == dx.dtype == torch.bfloat16 and dw.dtype == wdtype
    xq, xs, xqt, xst = tb.two_way_cast_to_fp8(x.detach())
    dq, ds, dqt, dst = tb.two_way_cast_to_fp8(dy)
    wq, ws, wqt, wst = tb.per_block_cast_to_fp8(w.detach().to(torch.bfloat16), transposed=True)
    _check(y.detach(), xq, xs, wq, ws)
    _check(dx, dq, ds, wqt, wst)
    _check(dw, dqt, dst, xqt, xst)


def test_linear_gradient_against_differences():
    """The layer is linear in dy and, for codes that do not move, in x: <dy, y(x + h) - y(x)> = <dx, h>
    for h that moves x from one set of exactly representable values to another."""
    g = torch.Generator().manual_seed(0)
    M, N, K = 32, 128, 256

    def exact(rows, cols, step):  # small integers times a power of two, a 448 in every group: codes are exact
        v = torch.randint(-8, 9, (rows, cols), generator=g).float() * 16
        v[:, ::128] = 448.0
        v[0, :] = 448.0
        return (v * step).to(torch.bfloat16).cuda()

    w = exact(N, K, 2.0**-6)
    dy = exact(M, N, 2.0**-9)
    x0, x1 = exact(M, K, 2.0**-4), exact(M, K, 2.0**-4)
    y0, y1 = tb.fp8_linear(x0, w), tb.fp8_linear(x1, w)
    x = x0.clone().requires_grad_()
    (dx,) = torch.autograd.grad(tb.fp8_linear(x, w), x, dy)
    left = (dy.double() * (y1.double() - y0.double())).sum()
    right = (dx.double() * (x1.double() - x0.double())).sum()
    # y and dx are rounded to bf16: 2^-9 of each of their magnitudes
    slack = 2.0**-8 * ((dy.double().abs() * (y1.double().abs() + y0.double().abs())).sum()
                       + (dx.double().abs() * (x1.double() - x0.double()).abs()).sum())
    assert abs(left - right) <= slack
    wv = w.clone().requires_grad_()
    (dw,) = torch.autograd.grad(tb.fp8_linear(x0, wv), wv, dy)
    w1 = exact(N, K, 2.0**-6)
    left = (dy.double() * (tb.fp8_linear(x0, w1).double() - y0.double())).sum()
    right = (dw.double() * (w1.double() - w.double())).sum()
    slack = 2.0**-8 * ((dy.double().abs() * (tb.fp8_linear(x0, w1).double().abs() + y0.double().abs())).sum()
                       + (dw.double().abs() * (w1.double() - w.double()).abs()).sum())
    assert abs(left - right) <= slack


def test_linear_with_cached_weight_leading_dimensions_and_partial_gradients():
    x = _matrix(60, 256, seed=1).cuda().reshape(3, 20, 256)
    w = _matrix(128, 256, seed=2, scale=0.02).cuda()
    cached = tb.per_block_cast_to_fp8(w, transposed=True)
    y = tb.fp8_linear(x, w, cached)
    assert y.shape == (3, 20, 128)
    assert torch.equal(y, tb.fp8_linear(x, w))
    assert torch.equal(y, tb.fp8_linear(x, w, (*cached[:2], None, None)))
    xg = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(tb.fp8_linear(xg, w, cached).sum(), xg)  # an expanded gradient
    (dx2,) = torch.autograd.grad(tb.fp8_linear(xg, w), xg, torch.ones_like(y))
    assert torch.equal(dx, dx2)
    wg = w.clone().requires_grad_()
    (dw,) = torch.autograd.grad(tb.fp8_linear(x, wg), wg, torch.ones_like(y))
    assert dw.shape == w.shape
    with pytest.raises(ValueError, match="transposed"):
        torch.autograd.grad(tb.fp8_linear(xg, w, (*cached[:2], None, None)), xg, torch.ones_like(y))
    with torch.no_grad():
        assert not tb.fp8_linear(xg, wg).requires_grad
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(tb.fp8_linear(xg, w), xg, torch.ones_like(y), create_graph=True)


def test_linear_without_tokens():
    x = torch.empty(0, 256, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    w = _matrix(128, 256, seed=2, scale=0.02).cuda().requires_grad_()
    y = tb.fp8_linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert dx.shape == (0, 256) and bool((dw == 0).all())


def test_linear_refusals():
    x = torch.zeros(4, 128, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(64, 128, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="bfloat16"):
        tb.fp8_linear(x.float(), w)
    with pytest.raises(ValueError, match="K"):
        tb.fp8_linear(x, w[:, :120])
    with pytest.raises(ValueError, match="multiples of 8"):
        tb.fp8_linear(x, w[:60])
    with pytest.raises(ValueError, match="float32"):
        tb.fp8_linear(x, w.half())


# Enough 256 x 256 tiles for pairs of CTAs: one round and a rest, the rest cut into
# 128 x 128 tiles (from 32 K blocks on), a last row tile with one CTA's rows only, a
# last column tile with half of its columns, odd columns and a short last K block.
PAIRS = [(2300, 2100, 300), (2300, 2304, 4200), (4737, 1025, 520), (2560, 2048, 128), (19000, 250, 1000)]


@pytest.mark.parametrize("kind", ["blocks", "rows"])
@pytest.mark.parametrize("M,N,K", PAIRS)
def test_product_of_many_tiles(M, N, K, kind):
    a, sa, b, sb = _operands(M, N, K, kind, seed=M + N + K)
    _check(tb.fp8_block_gemm(a, sa, b, sb), a, sa, b, sb)
    base = torch.randn(M, N, generator=torch.Generator().manual_seed(K)).cuda()
    d = base.clone()
    tb.fp8_block_gemm(a, sa, b, sb, out=d, accumulate=True)
    _check(d, a, sa, b, sb, base)
    again = base.clone()
    tb.fp8_block_gemm(a, sa, b, sb, out=again, accumulate=True)
    assert torch.equal(d, again)
