"""Gradients of any magnitude through fp8_linear, and the gradients' cast itself.

A loss averaged over many tokens gives gradients far below the activations' least scale
(1e-4, at which the codes of |dy| < 9.8e-8 are all zero), so a group of the incoming gradient
whose maximum is below 1e-4 has the scale max(amax / 448, 2^-92).

Tolerance against the unquantized gradient: e4m3 has 3 mantissa bits, a relative rounding error of
at most 2^-4 an element, 2^-4 / sqrt(3) in the mean square where values fill a binade evenly; a
product of two cast operands carries both (sqrt(2) 2^-4 / sqrt(3) = 0.051), and bf16's rounding.
"""

import pytest
import torch

import thingy_b200 as tb

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
FLOOR = 2.0**-92


def _normal(M, H, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(M, H, generator=g)


def _grads(x, w, dy):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    return torch.autograd.grad(tb.fp8_linear(x, w), (x, w), dy)


@pytest.mark.parametrize("wdtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("std", [1e-1, 1e-3, 1e-4, 4e-5, 2e-5, 1e-5, 1e-6, 1e-7, 1e-8, 1e-12, 1e-20])
def test_small_gradients_are_not_lost(std, wdtype):
    M, N, K = 300, 264, 392
    x = _normal(M, K, 1).to(torch.bfloat16).cuda()
    w = (0.05 * _normal(N, K, 2)).to(torch.bfloat16).to(wdtype).cuda()
    dy = (std * _normal(M, N, 3)).to(torch.bfloat16).cuda()
    dx, dw = _grads(x, w, dy)
    for got, want in ((dx, dy.double() @ w.double()), (dw, dy.double().t() @ x.double())):
        error = ((got.double() - want).norm() / want.norm()).item()
        assert error < 0.051 + 2.0**-9, error


@pytest.mark.parametrize("M,N,K", [(1, 128, 256), (40, 264, 136), (300, 520, 264)])
@pytest.mark.parametrize("shift", [4, 14, 24, 50])
def test_gradients_scale_with_the_incoming_one(M, N, K, shift):
    """2^-k dy has the same codes and 2^-k of the scales, so its gradients are 2^-k of dy's, bit for bit.
    dy is below 1e-4, and has no group whose scale 2^-92 would reach even at the last shift."""
    x = _normal(M, K, 4).to(torch.bfloat16).cuda()
    w = (0.05 * _normal(N, K, 5)).to(torch.bfloat16).cuda()
    dy = (2.0**-20 * _normal(M, N, 6)).to(torch.bfloat16).cuda()
    assert dy.abs().max() < 1e-4
    for got, want in zip(_grads(x, w, dy * 2.0**-shift), _grads(x, w, dy)):
        assert torch.equal(got, want * 2.0**-shift)


def test_cached_weight_and_one_orientation():
    x, w = _normal(20, 256, 7).to(torch.bfloat16).cuda(), (0.05 * _normal(136, 256, 8)).to(torch.bfloat16).cuda()
    dy = (1e-9 * _normal(20, 136, 9)).to(torch.bfloat16).cuda()
    want_dx, want_dw = _grads(x, w, dy)
    assert bool((want_dx != 0).any()) and bool((want_dw != 0).any())
    cached = tb.per_block_cast_to_fp8(w, transposed=True)
    xv, wv = x.clone().requires_grad_(), w.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(tb.fp8_linear(xv, w, cached), xv, dy)[0], want_dx)
    assert torch.equal(torch.autograd.grad(tb.fp8_linear(x, wv), wv, dy)[0], want_dw)


# ------------------------------------------------------------------ the cast


def _cast_ref(x, pow2):
    """Codes and scales of 1 x 128 groups on the CPU: division rounded to nearest even; the least scale is
    1e-4 where the group's maximum reaches it, else 2^-92."""
    x = x.float().cpu()
    R, C = x.shape
    full = torch.zeros(R, -(-C // 128) * 128)
    full[:, :C] = x
    amax = full.view(R, -1, 128).abs().amax(2)
    least = torch.where(amax < torch.tensor(1e-4), torch.tensor(FLOOR), torch.tensor(1e-4))
    s = torch.maximum(amax / 448.0, least)
    if pow2:
        m, e = torch.frexp(s)
        s = torch.ldexp(torch.ones_like(s), torch.where(m == 0.5, e - 1, e))
    return (x / s.repeat_interleave(128, 1)[:, :C]).to(F8), s


def _check_cast(x, pow2):
    q, s, qt, st = tb.two_way_cast_to_fp8(x.cuda(), pow2, gradient=True)
    for got_q, got_s, (want_q, want_s) in ((q, s, _cast_ref(x, pow2)), (qt, st, _cast_ref(x.t(), pow2))):
        assert torch.equal(got_s.cpu(), want_s)
        assert torch.equal(got_q.cpu().contiguous().view(torch.uint8), want_q.contiguous().view(torch.uint8))


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("scale", [1.0, 1e-4, 1e-7, 1e-12, 1e-20, 1e-25, 1e-26, 1e-28, 1e-30, 1e-36])
@pytest.mark.parametrize("M,H", [(1, 128), (130, 264)])
def test_gradient_cast(M, H, scale, pow2):
    """Down through the floor and to values that are zero at it, bit for bit."""
    x = scale * _normal(M, H, M + H)
    x[:, 3] = 0.0
    x[0, 5] = -0.0
    x[M - 1] *= 1e-3
    _check_cast(x.to(torch.bfloat16), pow2)


@pytest.mark.parametrize("pow2", [False, True])
def test_gradient_cast_of_every_maximum(pow2):
    """A row for every bf16 magnitude from 2^-85 to 2^-5 as its group's maximum, in each other elements
    spread over the codes' range."""
    bits = torch.arange((127 - 85) << 7, (127 - 5) << 7, dtype=torch.int32)
    top = (bits << 16).view(torch.float32)
    rest = torch.rand(len(top), 127, generator=torch.Generator().manual_seed(0)) * 2.0 ** torch.randint(
        -17, 1, (len(top), 127), generator=torch.Generator().manual_seed(1)).float()
    x = torch.cat([top[:, None], -top[:, None] * rest], dim=1)
    _check_cast(x.to(torch.bfloat16), pow2)


def test_activations_keep_their_floor():
    x = (1e-7 * _normal(40, 256, 3)).to(torch.bfloat16).cuda()
    for cast in (tb.two_way_cast_to_fp8(x), tb.two_way_cast_to_fp8(x, gradient=False)):
        floor = torch.tensor(1e-4, device="cuda")
        assert bool((cast[1] == floor).all()) and bool((cast[3] == floor).all())
    q, s, qt, st = tb.two_way_cast_to_fp8(x, gradient=True)
    assert bool((s < 1e-8).all()) and bool((q.float().abs().amax(1) == 448).all())


def test_gradients_of_at_least_1e_4_are_cast_as_activations():
    x = torch.randn(300, 264, generator=torch.Generator().manual_seed(4)) * 1e-2
    x[:, ::8] = 1e-3  # in every group along both axes
    x[::8] = 2e-4
    x = x.to(torch.bfloat16).cuda()
    for got, want in zip(tb.two_way_cast_to_fp8(x, gradient=True), tb.two_way_cast_to_fp8(x)):
        assert torch.equal(got.float(), want.float())


def test_gradient_cast_of_nonfinite_values():
    x = (1e-9 * _normal(130, 256, 2)).to(torch.bfloat16)
    x[1, 3] = float("nan")
    x[5, 200] = float("inf")
    q, s, qt, st = (t.float().cpu() for t in tb.two_way_cast_to_fp8(x.cuda(), gradient=True))
    assert torch.isnan(q[1, 3]) and torch.isnan(qt[3, 1]) and torch.isinf(s[5, 1]) and torch.isinf(st[200, 0])
    assert torch.isnan(q[5, 128:]).all() and torch.isnan(qt[200, :128]).all()
    assert int(torch.isnan(q).sum()) == 129 and int(torch.isnan(qt).sum()) == 129


def test_library_op_of_the_gradient_cast():
    import thingy_b200.custom_ops  # noqa: F401

    x = (1e-7 * _normal(40, 264, 5)).to(torch.bfloat16).cuda()
    op = torch.ops.thingy_b200.two_way_cast_to_fp8
    for gradient, got in ((True, op(x, False, True)), (False, op(x, False))):
        for a, b in zip(got, tb.two_way_cast_to_fp8(x, gradient=gradient)):
            assert a.stride() == b.stride() and torch.equal(a.float(), b.float())
    torch.library.opcheck(op, (x, False, True), test_utils="test_faketensor")
