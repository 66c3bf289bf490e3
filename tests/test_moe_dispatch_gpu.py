"""moe_sort, moe_permute and moe_combine against plain loops and 64-bit sums."""

import moe_reference as ref
import pytest
import torch

import thingy_b200 as tb

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounded_close(got, want, dtype, slack):
    """One rounding to dtype of a value within `slack` of `want`; below the normal range half the least spacing."""
    info = torch.finfo(dtype)
    tol = half_step(dtype) * (want.abs() + slack) + slack + info.tiny * info.eps
    off = (got.double().cpu() - want).abs()
    assert bool((off <= tol).all()), f"{float((off - tol).max())} over the tolerance"


def plan_of(T, k, E, align, seed, drop=0.0):
    ids = ref.choices(T, k, E, seed, drop)
    return tb.moe_sort(ids.cuda(), E, align=align), ref.sort(ids, E, align)


@pytest.mark.parametrize("align", [1, 16, 128])
@pytest.mark.parametrize("T,k,E,drop", [
    (0, 2, 8, 0.0), (1, 1, 1, 0.0), (1, 8, 128, 0.0), (3, 16, 512, 0.3), (64, 6, 64, 0.0), (511, 8, 60, 0.2),
    (512, 8, 256, 0.0), (513, 8, 33, 0.1),        # around the ids that one CTA sorts
    (2500, 3, 1, 0.0), (3001, 7, 512, 0.5), (20000, 8, 128, 0.1),
])
def test_sort_is_the_definition(T, k, E, drop, align):
    for dtype in (torch.int32, torch.int64):
        ids = ref.choices(T, k, E, 7 * T + E, drop, dtype)
        plan = tb.moe_sort(ids.cuda(), E, align=align)
        want = ref.sort(ids, E, align)
        assert plan.align == align
        for got, w in zip(plan[:4], want):
            assert got.dtype == torch.int32
            assert got.reshape(-1).tolist() == list(w)
        assert plan.positions.shape == (T, k)
        assert plan.sources.shape[0] == tb.moe_plan_rows(T, k, E, align)


def test_sort_of_many_chunks():
    """More chunks than one per 2048 choices: chunks grow."""
    T, k, E = 262144, 5, 200
    ids = ref.choices(T, k, E, 3, 0.05)
    plan, want = tb.moe_sort(ids.cuda(), E, align=128), ref.sort(ids, E, 128)
    for got, w in zip(plan[:4], want):
        assert torch.equal(got.reshape(-1).cpu(), torch.tensor(w, dtype=torch.int32))


@pytest.mark.parametrize("kind", ["one", "none", "last"])
def test_sort_of_lopsided_choices(kind):
    T, k, E = 3000, 4, 16
    value = {"one": 5, "none": -1, "last": E - 1}[kind]
    ids = torch.full((T, k), value, dtype=torch.int32)
    plan, want = tb.moe_sort(ids.cuda(), E, align=128), ref.sort(ids, E, 128)
    for got, w in zip(plan[:4], want):
        assert got.reshape(-1).tolist() == list(w)


def test_sort_of_strided_ids():
    ids = ref.choices(100, 8, 16, 1).cuda()
    plan, want = tb.moe_sort(ids.t().contiguous().t()[:, ::2], 16, align=1), tb.moe_sort(ids[:, ::2].contiguous(), 16, align=1)
    for a, b in zip(plan[:4], want[:4]):
        assert torch.equal(a, b)


ROWS = [(1, 1, 1, 1, 1, 0.0), (1, 8, 64, 128, 5120, 0.0), (3, 2, 4, 1, 7, 0.0), (33, 4, 16, 1, 1030, 0.3),
        (70, 16, 20, 16, 264, 0.2), (130, 9, 8, 128, 640, 0.0), (2500, 3, 8, 128, 72, 0.1), (5, 2, 3, 1, 33, 1.0),
        (0, 2, 4, 1, 64, 0.0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,align,H,drop", ROWS)
def test_permute_and_its_gradient(T, k, E, align, H, drop, dtype):
    plan, (sources, positions, _, _) = plan_of(T, k, E, align, 11, drop)
    g = torch.Generator().manual_seed(5)
    x = torch.randn(T, H, generator=g).to(dtype)
    R = len(sources)
    dxs = torch.randn(R, H, generator=g).to(dtype)
    xg = x.cuda().requires_grad_()
    xs = tb.moe_permute(xg, plan)
    assert torch.equal(xs.detach().double().cpu(), ref.permute(x, sources, k))
    (dx,) = torch.autograd.grad(xs, xg, dxs.cuda())
    terms = ref.gather(dxs, positions, T, k)
    assert dx.dtype == dtype and dx.shape == x.shape
    # k - 1 sums in fp32, each off by at most half a step of the terms' magnitudes
    rounded_close(dx, terms.sum(1), dtype, k * 2.0**-24 * terms.abs().sum(1))


@pytest.mark.parametrize("dtype", [torch.uint8, torch.float8_e4m3fn, torch.int32])
@pytest.mark.parametrize("H", [1, 40, 130, 7168])
def test_permute_of_codes_and_scales(dtype, H):
    T, k = 37, 5
    plan, (sources, _, _, _) = plan_of(T, k, 12, 128, 2, 0.2)
    raw = torch.randint(0, 256, (T, H * dtype.itemsize), generator=torch.Generator().manual_seed(1), dtype=torch.uint8)
    out = tb.moe_permute(raw.cuda().view(dtype), plan).view(torch.uint8).cpu()
    src = torch.tensor(sources)
    want = torch.where((src >= 0)[:, None], raw[src.clamp_min(0) // k], torch.zeros((), dtype=torch.uint8))
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,align,H,drop", ROWS)
def test_combine_and_its_gradients(T, k, E, align, H, drop, dtype):
    plan, (sources, positions, _, _) = plan_of(T, k, E, align, 13, drop)
    g = torch.Generator().manual_seed(6)
    R = len(sources)
    rows = torch.randn(R, H, generator=g).to(dtype)
    w = torch.rand(T, k, generator=g)
    dy = torch.randn(T, H, generator=g).to(dtype)
    rg, wg = rows.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = tb.moe_combine(rg, wg, plan)
    terms = w.double()[..., None] * ref.gather(rows, positions, T, k)
    assert y.dtype == dtype and y.shape == (T, H)
    rounded_close(y.detach(), terms.sum(1), dtype, k * 2.0**-24 * terms.abs().sum(1))
    drows, dw = torch.autograd.grad(y, (rg, wg), dy.cuda())
    src = torch.tensor(sources, dtype=torch.long)
    scale = torch.where(src >= 0, w.double().reshape(-1)[src.clamp_min(0)] if T else torch.zeros(R).double(), 0.0)
    want = scale[:, None] * (dy.double()[src.clamp_min(0) // k] if T else torch.zeros(R, H).double())
    rounded_close(drows, want, dtype, 2.0**-24 * want.abs())
    assert bool((drows[(src < 0).cuda()] == 0).all())
    dots = ref.gather(rows, positions, T, k) * dy.double()[:, None, :]
    off = (dw.double().cpu() - dots.sum(2)).abs()
    assert bool((off <= H * 2.0**-24 * dots.abs().sum(2)).all())  # H - 1 sums in some order
    # each gradient alone, the same bits
    assert torch.equal(torch.autograd.grad(tb.moe_combine(rg, w.cuda(), plan), rg, dy.cuda())[0], drows)
    assert torch.equal(torch.autograd.grad(tb.moe_combine(rows.cuda(), wg, plan), wg, dy.cuda())[0], dw)


def test_rows_of_other_strides():
    T, k, H = 50, 3, 96
    plan, _ = plan_of(T, k, 8, 1, 21)
    g = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.randn(T, 2 * H + 3, generator=g, device="cuda").bfloat16()
    for x in (wide[:, 1 : 1 + H], wide[:, 2 : 2 + 2 * H : 2], wide[:, 8 : 8 + H], wide[:1, :H].expand(T, H)):
        assert torch.equal(tb.moe_permute(x, plan), tb.moe_permute(x.contiguous(), plan))
    rows = torch.randn(T * k, 2 * H + 3, generator=g, device="cuda").bfloat16()
    w = torch.rand(k, T, generator=g, device="cuda").t()
    dy = torch.randn(H, T, generator=g, device="cuda").bfloat16().t()
    for r in (rows[:, 3 : 3 + H], rows[:, 1 : 1 + 2 * H : 2], rows[:, 2 : 2 + H]):
        a, b = r.detach().requires_grad_(), r.contiguous().requires_grad_()
        wa, wb = w.detach().requires_grad_(), w.contiguous().requires_grad_()
        ya, yb = tb.moe_combine(a, wa, plan), tb.moe_combine(b, wb, plan)
        assert torch.equal(ya, yb)
        ga = torch.autograd.grad(ya, (a, wa), dy)
        gb = torch.autograd.grad(yb, (b, wb), dy.contiguous())
        # other vectors, the same sums of a lane's elements only for rows: dw in another order
        assert torch.equal(ga[0], gb[0])
        assert torch.allclose(ga[1], gb[1], rtol=0, atol=float(H * 2.0**-24 * (dy.float().abs().sum(1).max() * r.abs().max())))


def test_rows_past_32_bits_of_offsets():
    """More than 2^31 elements of sorted rows: permute, combine and its backward at the far end."""
    T, k, H = 40000, 8, 7168
    ids = torch.arange(T * k, device="cuda", dtype=torch.int32).reshape(T, k) % 64
    plan = tb.moe_sort(ids, 64)
    assert plan.sources.numel() * H > 2**31
    x = torch.randint(-8, 8, (T, H), device="cuda", dtype=torch.int8, generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    xs = tb.moe_permute(x, plan)
    src = plan.sources.long()
    for r in (0, 1, 299999, T * k // 2, T * k - 2, T * k - 1):
        assert torch.equal(xs[r], x[src[r] // k])
    w = torch.full((T, k), 0.25, device="cuda")
    assert torch.equal(tb.moe_combine(xs, w, plan), 2 * x)  # small integers: exact in bf16
    wg, rg = w.requires_grad_(), xs.requires_grad_()
    drows, dw = torch.autograd.grad(tb.moe_combine(rg, wg, plan), (rg, wg), x)
    for r in (0, 299999, T * k - 1):
        assert torch.equal(drows[r], 0.25 * x[src[r] // k])
    assert torch.equal(dw, x.float().square().sum(1, keepdim=True).expand(T, k))  # integers below 2^24


def test_gradients_of_a_sum_and_of_broadcasts():
    """Gradients that come expanded (a sum's) and inputs used twice."""
    T, k, H = 20, 4, 48
    plan, (sources, positions, _, _) = plan_of(T, k, 6, 128, 3, 0.1)
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(3))
    xg = x.cuda().requires_grad_()
    w = torch.ones(T, k, device="cuda").requires_grad_()
    tb.moe_combine(tb.moe_permute(xg, plan), w, plan).sum().backward()
    made = (torch.tensor(positions).reshape(T, k) >= 0).double()
    assert torch.equal(xg.grad.double().cpu(), made.sum(1, keepdim=True).expand(T, H))
    off = (w.grad.double().cpu() - made * x.double().sum(1, keepdim=True)).abs()
    assert bool((off <= H * 2.0**-24 * x.double().abs().sum(1, keepdim=True)).all())


def test_infinities_and_nans_stay_in_their_tokens():
    T, k, H = 6, 2, 16
    ids = torch.tensor([[0, 1], [1, 2], [-1, 0], [-1, -1], [2, 1], [0, 2]], dtype=torch.int32)
    plan = tb.moe_sort(ids.cuda(), 3, align=128)
    rows = torch.randn(plan.sources.shape[0], H, device="cuda")
    rows[plan.sources < 0] = float("nan")  # padding is never read
    p = plan.positions.tolist()
    rows[p[0][0]] = float("inf")
    rows[p[4][1]] = float("nan")
    y = tb.moe_combine(rows, torch.full((T, k), 0.5, device="cuda"), plan).cpu()
    assert bool(torch.isinf(y[0]).all()) and bool(torch.isnan(y[4]).all())
    assert bool(torch.isfinite(y[[1, 2, 3, 5]]).all())
    assert bool((y[3] == 0).all())


def test_a_plan_out_of_range_reads_and_writes_nothing_there():
    T, k, H = 4, 2, 32
    positions = torch.tensor([[0, 99], [-7, 1], [2, 8], [3, 4]], dtype=torch.int32, device="cuda")
    sources = torch.tensor([0, 3, 4, 6, 7, -1, -1, -5], dtype=torch.int32, device="cuda")
    plan = tb.MoePlan(sources, positions, torch.zeros(2, dtype=torch.int32, device="cuda"),
                      torch.zeros(1, dtype=torch.int32, device="cuda"), 1)
    x = torch.randn(T, H, device="cuda")
    xs = tb.moe_permute(x, plan)
    assert torch.equal(xs, torch.cat([x[0:1], x[1:2], x[2:3], x[3:4], x[3:4], torch.zeros(3, H, device="cuda")]))
    y = tb.moe_combine(xs, torch.ones(T, k, device="cuda"), plan)
    assert torch.equal(y, torch.stack([x[0], x[1], x[2], x[3] + x[3]]))


def test_repeats_streams_and_graphs():
    """The same bits again, on another stream, and replayed from a graph with other inputs in the same places."""
    T, k, E, H = 700, 8, 64, 512
    ids = [ref.choices(T, k, E, s).cuda() for s in (1, 2)]
    x = [torch.randn(T, H, device="cuda").bfloat16() for _ in range(2)]
    w = torch.rand(T, k, device="cuda")

    def step(ids, x):
        plan = tb.moe_sort(ids, E, align=128)
        x = x.detach().requires_grad_()
        y = tb.moe_combine(tb.moe_permute(x, plan), w, plan)
        return (*plan[:4], y, torch.autograd.grad(y, x, torch.ones_like(y))[0])

    want = [[t.clone() for t in step(i, v)] for i, v in zip(ids, x)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a, b in zip(step(ids[0], x[0]), want[0]):
            assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(side)
    places = ids[0].clone(), x[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*places)
    for i in (1, 0, 1):
        places[0].copy_(ids[i]), places[1].copy_(x[i])
        graph.replay()
        for a, b in zip(got, want[i]):
            assert torch.equal(a, b)


def test_refusals():
    ids = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    plan = tb.moe_sort(ids, 4)
    x = torch.zeros(4, 8, device="cuda")
    w = torch.zeros(4, 2, device="cuda")
    rows = torch.zeros(8, 8, device="cuda")
    for call, match in [
        (lambda: tb.moe_sort(ids.cpu(), 4), "CUDA"),
        (lambda: tb.moe_sort(ids.float(), 4), "int32 or int64"),
        (lambda: tb.moe_sort(ids[0], 4), "2-D"),
        (lambda: tb.moe_sort(ids, 513), "512 experts"),
        (lambda: tb.moe_sort(ids, 0), "E, align > 0"),
        (lambda: tb.moe_sort(ids, 4, align=0), "E, align > 0"),
        (lambda: tb.moe_sort(ids, 4, align=65537), "align"),
        (lambda: tb.moe_sort(ids[:, :0], 4), "k, E"),
        (lambda: tb.moe_permute(x[:3], plan), "tokens"),
        (lambda: tb.moe_permute(x.double(), plan), "1, 2 or 4 bytes"),
        (lambda: tb.moe_permute(x.cpu(), plan), "CUDA"),
        (lambda: tb.moe_permute(x[:, :0], plan), "H > 0"),
        (lambda: tb.moe_permute(x, plan._replace(sources=plan.sources.long())), "sources"),
        (lambda: tb.moe_permute(x, plan._replace(positions=plan.positions.cpu())), "positions"),
        (lambda: tb.moe_combine(rows[:7], w, plan), "plan's 8 rows"),
        (lambda: tb.moe_combine(rows, w.bfloat16(), plan), "float32"),
        (lambda: tb.moe_combine(rows, w[:, :1], plan), "float32"),
        (lambda: tb.moe_combine(rows.to(torch.float8_e4m3fn), w, plan), "bfloat16, float16 or float32"),
        (lambda: tb.moe_combine(rows[:, :0], w, plan), "column"),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(tb.moe_permute(x, plan).sum(), x, create_graph=True)
