"""fp8_linear takes any layout of its tensors: each test compares a call whose input or
incoming gradient is laid out otherwise with the same call on a dense copy, bit for bit."""

import pytest
import torch

import thingy_b200 as tb

pytestmark = pytest.mark.gpu


def _matrix(M, H, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(M, H, generator=g)).to(torch.bfloat16).cuda()


def _step(x, w, dy=None):
    """y, dx and dw of one step; dx in x's own shape."""
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = tb.fp8_linear(x, w)
    return (y.detach(), *torch.autograd.grad(y, (x, w), torch.ones_like(y) if dy is None else dy))


def _same(got, want):
    for a, b in zip(got, want):
        assert a.shape == b.shape and torch.equal(a, b)


def _strided(kind):
    """A row of 256 elements (or a matrix of such rows) whose last dimension is not dense, in a
    storage large enough that a dense reading of it stays inside."""
    wide = _matrix(600, 600, seed=11)
    return {
        "column": lambda: wide[:256, 8],  # 1-D, stride 600
        "column as a row": lambda: wide.t()[8:9, :256],
        "stepped row": lambda: wide[:1, 0:512:2],
        "stepped row in three dimensions": lambda: wide[None, 8:9, 0:512:2],
        "rows of a transpose": lambda: wide.t()[8:40, :256],
        "stepped rows": lambda: wide[:40, 0:512:2],
        "rows off the 16-byte boundaries": lambda: wide[:40, 3:259],
    }[kind]()


@pytest.mark.parametrize("kind", ["column", "column as a row", "stepped row", "stepped row in three dimensions",
                                  "rows of a transpose", "stepped rows"])
def test_input_of_any_strides(kind):
    x, w = _strided(kind), _matrix(136, 256, seed=2, scale=0.02)
    assert x.stride(-1) != 1
    _same(_step(x, w), _step(x.contiguous(), w))


@pytest.mark.parametrize("shape", [(256,), (1, 256), (24, 256)])
def test_expanded_input(shape):
    """Broadcast inputs: nothing past their storage is read, and the gradient reaches them."""
    x, w = _matrix(1, 1, seed=3), _matrix(136, 256, seed=2, scale=0.02)
    wide = x.reshape(()).expand(shape)
    _same(_step(wide, w), _step(wide.contiguous(), w))
    row = _matrix(1, 256, seed=4)
    _same(_step(row.expand(24, 256), w), _step(row.expand(24, 256).contiguous(), w))


def test_weight_of_any_strides():
    x, wide = _matrix(24, 256, seed=3), _matrix(512, 512, seed=2, scale=0.02)
    for w in (wide.t()[:136, :256], wide[:136, 0:512:2], wide[:8, :256][:1].expand(8, 256)):
        _same(_step(x, w), _step(x, w.contiguous()))


def test_input_and_weight_off_the_16_byte_boundaries():
    x, w = _strided("rows off the 16-byte boundaries"), _matrix(136, 600, seed=2, scale=0.02)[:, 5:261]
    _same(_step(x, w), _step(x.contiguous(), w.contiguous()))
    flat = _matrix(1, 3 + 24 * 256, seed=5).view(-1)
    x = flat[3:].view(24, 256)
    assert x.is_contiguous() and x.data_ptr() % 16 != 0
    _same(_step(x, w), _step(x.clone(), w.contiguous()))


@pytest.mark.parametrize("rows", [1, 24])
def test_gradient_off_the_16_byte_boundaries(rows):
    """The gradient that autograd hands back for one part of a concatenation is a view into the whole."""
    x, w = _matrix(rows, 256, seed=3).requires_grad_(), _matrix(136, 256, seed=2, scale=0.02).requires_grad_()
    weight = _matrix(1, 3 + rows * 136, seed=6).view(-1)
    y = tb.fp8_linear(x, w)
    joined = torch.cat([torch.zeros(3, dtype=torch.bfloat16, device="cuda"), y.view(-1)])
    got = torch.autograd.grad(joined, (x, w), weight)
    _same(got, _step(x, w, weight[3:].clone().view(rows, 136))[1:])


@pytest.mark.parametrize("rows", [1, 24])
def test_gradient_of_any_strides(rows):
    x, w = _matrix(rows, 256, seed=3), _matrix(136, 256, seed=2, scale=0.02)
    wide = _matrix(600, 600, seed=7)
    for dy in (wide.t()[:rows, :136], wide[:rows, 0:272:2], wide[:1, :1].expand(rows, 136), wide[:1, :136].expand(rows, 136)):
        _same(_step(x, w, dy), _step(x, w, dy.contiguous()))


@pytest.mark.parametrize("M,N,K", [(24, 0, 256), (24, 136, 0), (0, 136, 256), (0, 0, 256), (24, 0, 0)])
def test_sizes_of_zero(M, N, K):
    """A sum over nothing is zero, and nothing has a gradient of its own shape."""
    x, w = torch.ones(M, K, dtype=torch.bfloat16, device="cuda"), torch.ones(N, K, dtype=torch.bfloat16, device="cuda")
    y, dx, dw = _step(x, w)
    assert y.shape == (M, N) and dx.shape == (M, K) and dw.shape == (N, K)
    for t in (y, dx, dw):
        assert bool((t == 0).all())


def _requested():
    """Bytes asked of the allocator and not given back, without its own rounding to blocks."""
    return torch.cuda.memory_stats()["requested_bytes.all.current"]


@pytest.mark.parametrize("wdtype", [torch.bfloat16, torch.float32])
def test_backward_holds_the_codes_that_it_reads(wdtype):
    """Between the passes a layer holds x's and the weight's codes along their columns, a byte an
    element and the scales, and nothing of the codes along the rows."""
    M, N, K = 2048, 768, 1024
    x, w = _matrix(M, K, seed=3).requires_grad_(), _matrix(N, K, seed=2, scale=0.02).to(wdtype).requires_grad_()
    tb.fp8_linear(x, w).sum().backward()  # what the library keeps for itself is there
    x.grad = w.grad = None
    torch.cuda.synchronize()
    before = _requested()
    y = tb.fp8_linear(x, w)
    held = _requested() - before
    codes = K * M + 4 * K * (M // 128) + K * N + 4 * (K // 128) * (N // 128)
    assert held <= y.numel() * 2 + codes + 3 * 512  # the layer's own alignment of its parts


@pytest.mark.parametrize("need_dx,need_dw,cached", [(True, False, False), (False, True, False), (True, True, True),
                                                    (True, False, True), (False, False, False)])
def test_backward_holds_no_more_than_its_gradients_need(need_dx, need_dw, cached):
    M, N, K = 2048, 768, 1024
    x, w = _matrix(M, K, seed=3).requires_grad_(need_dx), _matrix(N, K, seed=2, scale=0.02).requires_grad_(need_dw)
    codes = tb.per_block_cast_to_fp8(w.detach(), transposed=True) if cached else None
    dy = _matrix(M, N, seed=4, scale=0.1)
    want = _step(x, w, dy)
    torch.cuda.synchronize()
    before = _requested()
    y = tb.fp8_linear(x, w, codes)
    held = _requested() - before
    need = (K * M + 4 * K * (M // 128) if need_dw else 0) + (K * N + 4 * (K // 128) * (N // 128) if need_dx and not cached else 0)
    assert held <= y.numel() * 2 + need + 3 * 512
    wanted = [(t, g) for t, g, need_it in ((x, want[1], need_dx), (w, want[2], need_dw)) if need_it]
    assert torch.equal(y, want[0])
    if wanted:
        for got, (_, ref) in zip(torch.autograd.grad(y, [t for t, _ in wanted], dy), wanted):
            assert torch.equal(got, ref)
