"""The experts' products on sorted rows against 64-bit products of the dequantized operands, expert by expert.

Tolerances: the inner sum of a 128-wide block is fp32 in any order (at most
128 roundings of partial sums, each bounded by the sum of the magnitudes), two
roundings of the scales, one of the outer sum a block, then the output's.
"""

import moe_reference as ref
import pytest
import torch

import thingy_b200 as tb

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def spread(s, n, dim=-1):
    return s.double().repeat_interleave(128, dim).narrow(dim, 0, n)


def dequant_rows(q, s):
    return q.double() * spread(s, q.shape[1])


def dequant_blocks(q, s):
    return q.double() * spread(spread(s, q.shape[0], 0), q.shape[1])


def sum_error(K):
    """Of a sum of K products, in parts of the sum of their magnitudes."""
    return (130 + -(-K // 128)) * 2.0**-23


def check(got, a, b, out_dtype):
    """got = a @ b.T within the sums' and the output's rounding."""
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    eps = torch.finfo(out_dtype).eps / 2
    tol = sum_error(a.shape[1]) * size + eps * want.abs() + 1e-30
    assert bool(((got.double() - want).abs() <= tol).all())


def plan_of(counts, k=1, extra=0):
    """A plan whose experts have the given numbers of rows; `extra` choices are absent."""
    ids = torch.cat([torch.full((c,), e, dtype=torch.int32) for e, c in enumerate(counts)] +
                    [torch.full((extra,), -1, dtype=torch.int32)])
    ids = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(len(ids)))]
    return tb.moe_sort(ids.reshape(-1, k).cuda(), len(counts), align=128)


# the last three: few rows an expert in the mean, of which some have more than a kernel's 64 at a time
COUNTS = [[1], [128], [300, 0, 1, 127], [0, 0, 5], [129, 256, 0, 1000, 64], [0] * 9 + [513], [2000, 1],
          [7] * 40, [200] + [0] * 29 + [3], [64, 65, 16, 17, 0, 33, 1, 0, 48, 31] + [2] * 6]


def codes(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda").mul(60).clamp(-448, 448).to(F8)


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,K", [(16, 128), (128, 16), (256, 512), (640, 1040), (2064, 384), (304, 2064)])
@pytest.mark.parametrize("counts", COUNTS)
def test_product(counts, N, K, out_dtype):
    E, plan = len(counts), plan_of(counts, extra=70)
    R, KB = plan.sources.shape[0], -(-K // 128)
    g = torch.Generator(device="cuda").manual_seed(N + K)
    a, sa = codes(g, R, K), torch.rand(R, KB, generator=g, device="cuda") + 0.5
    a[plan.sources < 0] = torch.tensor(float("nan")).to(F8).cuda()
    b, sb = codes(g, E, N, K), torch.rand(E, -(-N // 128), KB, generator=g, device="cuda") + 0.5
    out = torch.full((R, N), float("nan"), dtype=out_dtype, device="cuda")
    got = tb.fp8_grouped_gemm(a, sa, b, sb, plan, out=out)
    assert got.data_ptr() == out.data_ptr()
    off = plan.offsets.tolist()
    for e in range(E):
        rows = slice(off[e], off[e + 1])
        check(got[rows][: counts[e]], dequant_rows(a[rows], sa[rows])[: counts[e]], dequant_blocks(b[e], sb[e]), out_dtype)
    assert bool((got[plan.sources < 0] == 0).all())  # whatever a holds there
    # scales in the other order, another stride of the experts, the same bits
    wide = torch.zeros(E, N + 3, K, dtype=F8, device="cuda")
    wide[:, :N] = b
    again = tb.fp8_grouped_gemm(a, sa.t().contiguous().t(), wide[:, :N], sb.transpose(1, 2).contiguous().transpose(1, 2), plan,
                                out_dtype=out_dtype)
    assert torch.equal(again, got)


@pytest.mark.parametrize("counts", [[300, 0, 1, 127], [7] * 40])  # either kernel
def test_operands_of_other_strides(counts):
    """Rows of A and D inside wider ones, one matrix for all experts: the same bits; off the boundaries: refused."""
    E, plan, N, K = len(counts), plan_of(counts), 256, 384
    R = plan.sources.shape[0]
    g = torch.Generator(device="cuda").manual_seed(8)
    a, sa = codes(g, R, K), torch.rand(R, 3, generator=g, device="cuda")
    b, sb = codes(g, 1, N, K), torch.rand(1, 2, 3, generator=g, device="cuda")
    want = tb.fp8_grouped_gemm(a, sa, b.expand(E, N, K).contiguous(), sb.expand(E, 2, 3).contiguous(), plan)
    wide = torch.zeros(R, K + 48, dtype=F8, device="cuda")
    wide[:, 16 : 16 + K] = a
    out = torch.full((R, N + 32), 7.0, dtype=torch.bfloat16, device="cuda")
    got = tb.fp8_grouped_gemm(wide[:, 16 : 16 + K], sa, b.expand(E, N, K), sb.expand(E, 2, 3), plan, out=out[:, 16 : 16 + N])
    assert torch.equal(got, want)
    assert bool((out[:, :16] == 7).all()) and bool((out[:, 16 + N :] == 7).all())
    for bad in (wide[:, 8 : 8 + K], wide.view(torch.uint8)[:, 1 : 1 + K]):
        with pytest.raises(ValueError, match="aligned"):
            tb.fp8_grouped_gemm(bad, sa, b.expand(E, N, K), sb.expand(E, 2, 3), plan)
    with pytest.raises(ValueError, match="aligned"):
        tb.fp8_grouped_gemm(a, sa, b.expand(E, N, K), sb.expand(E, 2, 3), plan, out=out[:, 8 : 8 + N])


def test_product_equals_the_single_one():
    """An expert alone: the same tiles, the same sums as fp8_block_gemm over its rows."""
    counts = [384, 1, 200]
    plan = plan_of(counts)
    R, N, K, E = plan.sources.shape[0], 1024, 2048, 3
    g = torch.Generator(device="cuda").manual_seed(4)
    a, sa = codes(g, R, K), torch.rand(R, K // 128, generator=g, device="cuda")
    b, sb = codes(g, E, N, K), torch.rand(E, N // 128, K // 128, generator=g, device="cuda")
    got = tb.fp8_grouped_gemm(a, sa, b, sb, plan, out_dtype=torch.float32)
    off = plan.offsets.tolist()
    for e in range(E):
        rows = slice(off[e], off[e] + counts[e])
        want = tb.fp8_block_gemm(a[rows], sa[rows], b[e], sb[e], out_dtype=torch.float32)
        size = dequant_rows(a[rows], sa[rows]).abs() @ dequant_blocks(b[e], sb[e]).abs().t()
        assert bool(((got[rows] - want).double().abs() <= 2 * sum_error(K) * size).all())  # other forms there, K may be split


@pytest.mark.parametrize("R", [384, 512])  # the kernel for few rows an expert, and the other
def test_offsets_are_cut_to_the_rows(R):
    """Offsets out of range, decreasing or off the blocks: nothing is read or written outside."""
    N, K = 256, 256
    g = torch.Generator(device="cuda").manual_seed(2)
    a, sa = codes(g, R, K), torch.ones(R, 2, device="cuda")
    b, sb = codes(g, 3, N, K), torch.ones(3, 2, 2, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    lists = [0, 128, 900, 5000], [-300, 128, 0, 512], [0, 100, 300, 511], [512, 512, 512, 512], [0, 0, 0, 0]
    for values, n in [(v, n) for v in lists for n in ([1 << 30, -5, 200], [1, 2, 3])]:
        counts = torch.tensor(n, dtype=torch.int32, device="cuda")
        offsets = torch.tensor(values, dtype=torch.int32, device="cuda")
        guard = torch.full((R + 256, N), 7.0, device="cuda")
        tb.fp8_grouped_gemm(a, sa, b, sb, tb.MoePlan(none, none, offsets, counts, 128), out=guard[128 : 128 + R])
        assert bool((guard[:128] == 7).all()) and bool((guard[128 + R :] == 7).all())
        assert tb._lib.device_error() == 0


def quantized(x, rows, cols, gradient=False):
    """What x stands for on e4m3 codes in tiles of rows x cols (in fp32 as the casts make them)."""
    R, C = x.shape
    t = x.float().reshape(R // rows, rows, C // cols, cols)
    amax = t.abs().amax((1, 3), keepdim=True)
    s = amax / torch.full_like(amax, 448.0)
    s = torch.where(amax < 1e-4, s.clamp_min(2.0**-92), s.clamp_min(1e-4)) if gradient else s.clamp_min(1e-4)
    return ((t / s).to(F8).double() * s.double()).reshape(R, C)


@pytest.mark.parametrize("weight_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,K", [(128, 128), (384, 256), (1024, 640), (2048, 2048)])
@pytest.mark.parametrize("counts", [[1], [300, 0, 1, 127], [129, 256, 0, 1000, 64], [7] * 20, [100, 0, 2, 1, 9]])
def test_linear_and_gradients(counts, N, K, weight_dtype):
    E, plan = len(counts), plan_of(counts, extra=33)
    R = plan.sources.shape[0]
    g = torch.Generator(device="cuda").manual_seed(N * 3 + K)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    x, dy = rand(R, K).bfloat16(), (0.1 * rand(R, N)).bfloat16()
    pad = plan.sources < 0
    x[pad], dy[pad] = float("nan"), float("inf")  # padding counts as zeros, whatever it holds
    w = (0.02 * rand(E, N, K)).to(weight_dtype)
    xg, wg = x.requires_grad_(), w.requires_grad_()
    y = tb.fp8_grouped_linear(xg, wg, plan)
    dx, dw = torch.autograd.grad(y, (xg, wg), dy)
    assert y.dtype == dx.dtype == torch.bfloat16 and dw.dtype == weight_dtype
    assert y.shape == (R, N) and dx.shape == x.shape and dw.shape == w.shape
    x0, dy0 = x.detach().masked_fill(pad[:, None], 0), dy.masked_fill(pad[:, None], 0)
    off = plan.offsets.tolist()
    for e in range(E):
        rows = slice(off[e], off[e + 1])
        if not counts[e]:
            assert bool((dw[e] == 0).all())
            continue
        we = quantized(w[e].detach().bfloat16(), 128, 128)
        check(y[rows].detach(), quantized(x0[rows], 1, 128), we, torch.bfloat16)
        check(dx[rows], quantized(dy0[rows], 1, 128, True), we.t(), torch.bfloat16)
        check(dw[e], quantized(dy0[rows], 128, 1, True).t(), quantized(x0[rows], 128, 1).t(), weight_dtype)
    for t in (y.detach(), dx):
        assert bool((t[pad] == 0).all())
    # a cast made once, each gradient alone, other strides: the same bits
    cast = tb.quantize_experts(w.detach().bfloat16(), transposed=True)
    y2 = tb.fp8_grouped_linear(xg, wg, plan, cast)
    dx2, dw2 = torch.autograd.grad(y2, (xg, wg), dy)
    assert torch.equal(y2, y) and torch.equal(dx2, dx) and torch.equal(dw2, dw)
    assert torch.equal(torch.autograd.grad(tb.fp8_grouped_linear(xg, w.detach(), plan), xg, dy)[0], dx)
    wide = torch.zeros(R, N + 5, dtype=torch.bfloat16, device="cuda")
    wide[:, 3 : 3 + N] = dy
    xt = x.detach().t().contiguous().t()
    assert torch.equal(torch.autograd.grad(tb.fp8_grouped_linear(xt, wg, plan), wg, wide[:, 3 : 3 + N])[0], dw)
    with torch.no_grad():
        assert torch.equal(tb.fp8_grouped_linear(xg, wg, plan, (*cast[:2], None, None)), y)


def test_linear_against_differences():
    """The weight's gradient of a sum against differences of the layer, at steps that codes resolve.

    x and dy are powers of two: codes hold them exactly, so y is linear in a weight while its block's scale stays."""
    plan = plan_of([100, 60])
    R, N, K = plan.sources.shape[0], 128, 128
    g = torch.Generator(device="cuda").manual_seed(5)
    made = (plan.sources >= 0)[:, None]
    x = torch.where(made, 2.0 ** torch.randint(-1, 2, (R, K), generator=g, device="cuda"), 0.0).bfloat16()
    w = torch.zeros(2, N, K, device="cuda")
    w[:, 0, 0] = 448.0  # the block's scale is one
    w[:, 1:, 1:] = torch.randint(-4, 5, (2, N - 1, K - 1), generator=g, device="cuda").float()
    wg = w.clone().requires_grad_()
    dy = torch.where(made, 2.0 ** torch.randint(-1, 2, (R, N), generator=g, device="cuda"), 0.0).bfloat16()

    def loss(weight):
        with torch.no_grad():
            return float((tb.fp8_grouped_linear(x, weight, plan).double() * dy.double()).sum())

    (dw,) = torch.autograd.grad(tb.fp8_grouped_linear(x, wg, plan), wg, dy)
    for e, n, k in [(0, 3, 5), (0, 127, 127), (1, 1, 90), (1, 64, 2)]:
        up, down = w.clone(), w.clone()
        up[e, n, k] += 1.0
        down[e, n, k] -= 1.0
        # y is rounded to bf16: a step of at most 2^-8 of |y| on each of the expert's rows, twice
        y = tb.fp8_grouped_linear(x, w, plan).double().abs() + 2.0
        tol = float((y * dy.double().abs())[:, n].sum()) * 2.0**-8
        assert abs((loss(up) - loss(down)) / 2 - float(dw[e, n, k])) <= tol


def test_one_weight_for_all_experts():
    """A weight that is expanded over the experts: its gradient is the sum of theirs."""
    plan = plan_of([100, 60, 0, 200])
    R = plan.sources.shape[0]
    g = torch.Generator(device="cuda").manual_seed(12)
    x = torch.randn(R, 256, generator=g, device="cuda").bfloat16()
    dy = torch.randn(R, 128, generator=g, device="cuda").bfloat16()
    one = (0.05 * torch.randn(1, 128, 256, generator=g, device="cuda")).requires_grad_()
    each = one.detach().expand(4, 128, 256).contiguous().requires_grad_()
    y = tb.fp8_grouped_linear(x, one.expand(4, 128, 256), plan)
    assert torch.equal(y, tb.fp8_grouped_linear(x, each, plan))
    (d1,) = torch.autograd.grad(y, one, dy)
    (d4,) = torch.autograd.grad(tb.fp8_grouped_linear(x, each, plan), each, dy)
    assert torch.equal(d1, d4.sum(0, keepdim=True))


def test_no_rows():
    plan = tb.moe_sort(torch.zeros(0, 2, dtype=torch.int32, device="cuda"), 4, align=128)
    x = torch.zeros(0, 128, dtype=torch.bfloat16, device="cuda").requires_grad_()
    w = torch.randn(4, 256, 128, device="cuda").requires_grad_()
    y = tb.fp8_grouped_linear(x, w, plan)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == (0, 256) and dx.shape == (0, 128) and bool((dw == 0).all())
    absent = tb.moe_sort(torch.full((3, 2), -1, dtype=torch.int32, device="cuda"), 4, align=128)
    x = torch.randn(absent.sources.shape[0], 128, device="cuda").bfloat16().requires_grad_()
    y = tb.fp8_grouped_linear(x, w, absent)
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert all(bool((t == 0).all()) for t in (y, dx, dw))


@pytest.mark.parametrize("counts", [[700, 300], [5, 20]])
def test_wait_limit(counts):
    """A wait that gives up ends the launch with a device error; the next one is whole."""
    plan = plan_of(counts)
    R, N, K = plan.sources.shape[0], 512, 2048
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(R, K, generator=g, device="cuda").bfloat16().requires_grad_()
    w = (0.02 * torch.randn(2, N, K, generator=g, device="cuda")).bfloat16().requires_grad_()
    dy = torch.randn(R, N, generator=g, device="cuda").bfloat16()

    def step():
        y = tb.fp8_grouped_linear(x, w, plan)
        return y.detach(), *torch.autograd.grad(y, (x, w), dy)

    want = step()
    q, s, _, _ = tb.two_way_cast_to_fp8(x.detach())
    b, sb = tb.quantize_experts(w.detach())
    torch.cuda.synchronize()
    tb._lib.device_error()
    old = tb._lib.set_wait_limit(-1)
    try:
        tb.fp8_grouped_gemm(q, s, b, sb, plan)
        torch.cuda.synchronize()
    finally:
        tb._lib.set_wait_limit(old)
    assert tb._lib.device_error() == 1
    assert tb._lib.device_error() == 0
    for a, b in zip(step(), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("N,K", [(2048, 2048), (256, 128)])  # pairs, and 128-wide tiles
def test_wait_limit_of_the_weight_gradient(N, K):
    """The same for the gradient, an expert without rows among them."""
    counts = [700, 0, 300, 64]
    plan = plan_of(counts)
    R, E = plan.sources.shape[0], len(counts)
    g = torch.Generator(device="cuda").manual_seed(10)
    a, b = codes(g, N, R), codes(g, K, R)
    sa, sb = torch.rand(N, R // 128, generator=g, device="cuda"), torch.rand(K, R // 128, generator=g, device="cuda")
    d = torch.zeros(E, N, K, device="cuda")
    lib = tb._lib.load()

    def launch():
        tb._lib.check(lib.cutie_fp8_grouped_wgrad(
            a.data_ptr(), R, sa.data_ptr(), R // 128, 1, b.data_ptr(), R, sb.data_ptr(), R // 128, 1, plan.offsets.data_ptr(), E,
            d.data_ptr(), K, N * K, tb._lib.DTYPE_F32, R, N, K, torch.cuda.current_stream().cuda_stream))
        return d.clone()

    want = launch()
    off = plan.offsets.tolist()
    for e in range(E):
        cols = slice(off[e], off[e + 1])
        left, right = (q[:, cols].double() * spread(s[:, off[e] // 128 : off[e + 1] // 128], off[e + 1] - off[e])
                       for q, s in ((a, sa), (b, sb)))
        check(want[e], left, right, torch.float32)
    torch.cuda.synchronize()
    tb._lib.device_error()
    old = tb._lib.set_wait_limit(-1)
    try:
        launch()
        torch.cuda.synchronize()
    finally:
        tb._lib.set_wait_limit(old)
    assert tb._lib.device_error() == 1
    assert torch.equal(launch(), want) and tb._lib.device_error() == 0


def test_repeats_and_graphs():
    E, N, K, T, k = 8, 256, 384, 300, 2
    g = torch.Generator(device="cuda").manual_seed(3)
    w = (0.02 * torch.randn(E, N, K, generator=g, device="cuda")).bfloat16()
    x = [torch.randn(T, K, generator=g, device="cuda").bfloat16() for _ in range(2)]
    ids = [ref.choices(T, k, E, s, 0.1).cuda() for s in (1, 2)]
    weights = torch.rand(T, k, generator=g, device="cuda")

    def step(x, ids):
        x, wg = x.detach().requires_grad_(), w.detach().requires_grad_()
        plan = tb.moe_sort(ids, E, align=128)
        y = tb.moe_combine(tb.fp8_grouped_linear(tb.moe_permute(x, plan), wg, plan), weights, plan)
        return y.detach(), *torch.autograd.grad(y, (x, wg), torch.ones_like(y))

    want = [[t.clone() for t in step(*a)] for a in zip(x, ids)]
    places = x[0].clone(), ids[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*places)
    for i in (1, 0, 1):
        places[0].copy_(x[i]), places[1].copy_(ids[i])
        graph.replay()
        for a, b in zip(got, want[i]):
            assert torch.equal(a, b)


def test_refusals():
    plan = plan_of([100, 60])
    R = plan.sources.shape[0]
    x = torch.zeros(R, 128, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(2, 256, 128, dtype=torch.bfloat16, device="cuda")
    a, sa = x.to(F8), torch.ones(R, 1, device="cuda")
    b, sb = w.to(F8), torch.ones(2, 2, 1, device="cuda")
    loose = tb.moe_sort(torch.zeros(4, 1, dtype=torch.int32, device="cuda"), 2, align=64)
    for call, match in [
        (lambda: tb.fp8_grouped_linear(x, w, loose), "multiple of 128"),
        (lambda: tb.fp8_grouped_linear(x[:-128], w, plan), "plan's"),
        (lambda: tb.fp8_grouped_linear(x.float(), w, plan), "bfloat16"),
        (lambda: tb.fp8_grouped_linear(x, w.half(), plan), "bfloat16 or float32"),
        (lambda: tb.fp8_grouped_linear(x, w[:, :200], plan), "multiples of 128"),
        (lambda: tb.fp8_grouped_linear(x, w[:1], plan), "E = 1"),
        (lambda: tb.fp8_grouped_linear(x, w.cpu(), plan), "wrong device"),
        (lambda: tb.fp8_grouped_linear(x, w[0], plan), "E, N, K"),
        (lambda: tb.fp8_grouped_linear(x.requires_grad_(), w, plan, (b, sb, None, None)), "transposed"),
        (lambda: tb.fp8_grouped_linear(x, w, plan, (b, sb, b, sb)), "transposes"),
        (lambda: tb.fp8_grouped_linear(x.detach(), w, plan, (b[:1], sb, None, None)), "weight_fp8"),
        (lambda: tb.fp8_grouped_gemm(a, sa, b, sb, loose), "multiple of 128"),
        (lambda: tb.fp8_grouped_gemm(a[:-1], sa[:-1], b, sb, plan), "multiples of 128"),
        (lambda: tb.fp8_grouped_gemm(a, sa[:, :0], b, sb, plan), "a_scale"),
        (lambda: tb.fp8_grouped_gemm(a, sa, b, sb[:, :1], plan), "scales"),
        (lambda: tb.fp8_grouped_gemm(a, sa, b[:, :, :112], sb, plan), "shape"),
        (lambda: tb.fp8_grouped_gemm(a, sa, b[:, :8], sb[:, :1], plan), "multiple of 16"),
        (lambda: tb.fp8_grouped_gemm(a, sa, b, sb, plan, out=torch.empty(R, 128, device="cuda")), "shape"),
        (lambda: tb.fp8_grouped_gemm(a, sa, b, sb, plan, out_dtype=torch.float16), "out_dtype"),
        (lambda: tb.fp8_grouped_gemm(a, sa, b, sb, plan, out=torch.empty(R, 257, device="cuda")[:, 1:]), "aligned"),
        (lambda: tb.fp8_grouped_gemm(a.t().contiguous().t(), sa, b, sb, plan), "contiguous"),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
