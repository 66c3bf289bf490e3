"""fp8_linear's gradients against differences that the tolerance resolves.

Operands are small integers times a power of two, with a 448 in every group at
a place that does not move, so every cast is exact, also of the moved operand,
and y is linear in each of them up to its rounding to bf16. The move h of an
operand takes the sign of its gradient element by element, so nothing in
<gradient, h> cancels: the rounding of the two y (2^-9 of each element) and of
the gradient (2^-9) is then a small part of it, and a gradient of zero, or of
the wrong sign, is outside.
"""

import pytest
import torch

import thingy_b200 as tb

pytestmark = pytest.mark.gpu
MOVE = 16.0


def _exact(g, rows, cols, step):
    """Multiples of 16 up to 128, so that one more step is a code too (four significant bits); 448 in
    one row and one column of every 128."""
    v = MOVE * torch.randint(-8, 9, (rows, cols), generator=g).float()
    v[:, ::128] = 448.0
    v[::128, :] = 448.0
    return (v * step).to(torch.bfloat16).cuda()


def _moved(t, sign, step):
    """t one step along the signs, where it is not one of the 448s; also the move."""
    h = MOVE * step * sign.float()
    h[:, ::128] = 0.0
    h[::128, :] = 0.0
    return (t.float() + h).to(torch.bfloat16), h


def _compare(grad, h, dy, y0, y1):
    left = (dy.double() * (y1.double() - y0.double())).sum().item()
    right = (grad.double() * h.double()).sum().item()
    slack = 2.0**-9 * ((dy.double().abs() * (y1.double().abs() + y0.double().abs())).sum()
                       + (grad.double().abs() * h.double().abs()).sum()).item()
    assert right > 0 and slack < 0.1 * right, (slack, right)
    assert abs(left - right) <= slack, (left, right, slack)
    for wrong in (0.0, -1.0, 2.0):  # what a missing, negated or doubled gradient would give
        assert abs(left - wrong * right) > slack


@pytest.mark.parametrize("M,N,K", [(32, 128, 256), (1, 128, 256), (200, 264, 136), (65, 384, 640)])
def test_gradients_against_differences(M, N, K):
    g = torch.Generator().manual_seed(M + N + K)
    sx, sw, sd = 2.0**-4, 2.0**-6, 2.0**-9
    x, w, dy = _exact(g, M, K, sx), _exact(g, N, K, sw), _exact(g, M, N, sd)
    if M == 1:  # the first row is not all the same here: one 448 a group holds the scale
        row = MOVE * torch.randint(-8, 9, (1, K), generator=g).float()
        row[:, ::128] = 448.0
        x = (row * sx).to(torch.bfloat16).cuda()
    xv, wv = x.clone().requires_grad_(), w.clone().requires_grad_()
    y0 = tb.fp8_linear(xv, wv)
    dx, dw = torch.autograd.grad(y0, (xv, wv), dy)
    y0 = y0.detach()
    if M > 1:
        x1, h = _moved(x, torch.sign(dx), sx)
        _compare(dx, h, dy, y0, tb.fp8_linear(x1, w))
    else:
        h = MOVE * sx * torch.sign(dx).float()
        h[:, ::128] = 0.0
        _compare(dx, h, dy, y0, tb.fp8_linear((x.float() + h).to(torch.bfloat16), w))
    w1, h = _moved(w, torch.sign(dw), sw)
    _compare(dw, h, dy, y0, tb.fp8_linear(x, w1))
