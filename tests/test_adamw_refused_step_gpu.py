"""A step that AdamW refuses does not count: parameters that were not stepped keep their number of steps."""

import pytest
import torch

import thingy_b200 as tb

pytestmark = pytest.mark.gpu


def steps_of(opt, params):
    return [int(opt.state[p]["step"]) for p in params]


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("before", [0, 2])
def test_refused_and_taken_again(before, capturable, bits):
    """A clip factor of a wrong type, then the right one: the same bits as without the refused call."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    start = [torch.randn(300, generator=gen, device="cuda"), torch.randn(129, generator=gen, device="cuda").bfloat16()]
    grads = [[torch.randn(p.shape, generator=gen, device="cuda").to(p.dtype) for p in start] for _ in range(before + 2)]
    clip = torch.full((1,), 0.5, device="cuda")
    results = []
    for refused in (False, True):
        params = [p.clone().requires_grad_() for p in start]
        opt = tb.AdamW(params, lr=0.1, state_bits=bits, capturable=capturable, seed=4)
        for t, gs in enumerate(grads):
            for p, g in zip(params, gs):
                p.grad = g.clone()
            if refused and t == before:
                old = [p.detach().clone() for p in params]
                for bad in (clip.double(), clip.cpu(), torch.ones(2, device="cuda")):
                    with pytest.raises(ValueError, match="grad_scale"):
                        opt.step(grad_scale=bad)
                    assert steps_of(opt, params) == [before, before]
                assert all(torch.equal(p, q) for p, q in zip(params, old))
            opt.step(grad_scale=clip)
        assert steps_of(opt, params) == [before + 2, before + 2]
        results.append(params)
    assert all(torch.equal(p, q) for p, q in zip(*results))


@pytest.mark.parametrize("capturable", [False, True])
def test_a_part_of_the_parameters_is_refused(capturable):
    """Lists that were stepped before the refusal have counted, the others not; all go on from there."""
    good = torch.randn(40, device="cuda", requires_grad=True)
    bad = torch.randn(8, 6, device="cuda").bfloat16().t().requires_grad_()  # not contiguous
    opt = tb.AdamW([good, bad], lr=0.1, capturable=capturable)
    for p in (good, bad):
        p.grad = torch.ones_like(p)
    for t in (1, 2):
        with pytest.raises(ValueError, match="contiguous"):
            opt.step()
        assert steps_of(opt, [good, bad]) == [t, 0]
    bad.data = bad.data.contiguous()
    bad.grad = torch.ones_like(bad)
    opt.step()
    assert steps_of(opt, [good, bad]) == [3, 1]
