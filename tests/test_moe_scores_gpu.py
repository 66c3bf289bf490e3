"""The experts' weights where their scores leave fp32's range and where a logit is a NaN, and the order of
what CTAs write for one another.

Reference in 64 bits, where the scores below do not underflow. The router's logits come from
one column, x[t, 0] router[e, 0] with x[t, 0] = 1, so they are the same numbers in both.
"""

import pytest
import torch

import thingy_b200 as tb
from thingy_b200.moe import quantize_experts

pytestmark = pytest.mark.gpu


def _layer(T, E, logits, seed, H=256, I=128):
    """Operands whose router gives `logits` [E] to every token (its first column alone is not zero)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    q, s, _, n = tb.rms_norm_fp8(x, torch.ones(H, dtype=torch.bfloat16, device="cuda"), 1e-6, return_normalized=True)
    n = n.clone()
    n[:, 0] = 1.0
    router = torch.zeros(E, H, device="cuda")
    router[:, 0] = logits
    w13 = quantize_experts((0.05 * torch.randn(E, 2 * I, H, generator=g, device="cuda")).to(torch.bfloat16))
    w2 = quantize_experts((0.05 * torch.randn(E, H, I, generator=g, device="cuda")).to(torch.bfloat16))
    return n, q, s, router.to(torch.bfloat16), *w13, *w2


def _call(ops, k, **kw):
    T = ops[0].shape[0]
    ids = torch.full((T, k), -1, dtype=torch.int32, device="cuda")
    weights = torch.full((T, k), -1.0, device="cuda")
    return tb.moe_fp8(*ops, top_k=k, topk_ids=ids, topk_weights=weights, **kw), ids.long(), weights.double()


def _scores(logits, scoring):
    return torch.softmax(logits, -1) if scoring == "softmax" else torch.sigmoid(logits)


@pytest.mark.parametrize("T", [1, 3, 20])
@pytest.mark.parametrize("base", [-50.0, -70.0, -95.0, -300.0, -30000.0])
def test_sigmoid_of_far_negative_logits(T, base):
    """Every chosen score below the least fp32 number: the weights are their ratios all the same."""
    steps = torch.tensor([0.0, 0.5, -0.5, -2.0, -4.0, -8.0, -1.0, -3.0], device="cuda")
    # the logits as bf16 holds them, apart by exact multiples of its step there
    unit = max(1.0, 2.0 ** (torch.tensor(-base).log2().floor().item() - 7))
    ops = _layer(T, 8, base + steps * unit * 2, seed=1)
    y, ids, weights = _call(ops, 3, scoring="sigmoid")
    logits = ops[3][:, 0].double()
    top = torch.sort(logits, descending=True, stable=True)
    # exp(l) / (1 + exp(l)) relative to the largest one, which 64 bits hold for any base
    want = torch.exp(top.values[:3] - top.values[0]) * (1 + torch.exp(top.values[0])) / (1 + torch.exp(top.values[:3]))
    assert torch.equal(ids, top.indices[:3].expand(T, 3))
    assert torch.allclose(weights, (want / want.sum()).expand(T, 3), rtol=1e-4, atol=1e-35)
    assert bool(torch.isfinite(y).all()) and bool((y != 0).any())


@pytest.mark.parametrize("T", [2, 20])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("low", [-40.0, -100.0, -160.0])
def test_bias_that_picks_experts_of_low_scores(T, scoring, low):
    logits = torch.tensor([4.0, 3.0, low, low + 1.0, low + 2.0, 0.0, 1.0, 2.0], device="cuda")
    ops = _layer(T, 8, logits, seed=2)
    bias = torch.zeros(8, device="cuda")
    bias[2:5] = torch.tensor([5.0, 4.0, 3.0])
    y, ids, weights = _call(ops, 3, scoring=scoring, bias=bias)
    assert torch.equal(ids, torch.tensor([2, 3, 4], device="cuda").expand(T, 3))
    p = _scores(ops[3][:, 0].double(), scoring)[2:5]
    assert torch.allclose(weights, (p / p.sum()).expand(T, 3), rtol=1e-4, atol=1e-35)
    assert bool(torch.isfinite(y).all()) and bool((y != 0).any())


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_scores_that_are_not_renormalized_may_be_zero(scoring):
    ops = _layer(3, 8, torch.tensor([2.0, 1.0, -300.0, -301.0, -302.0, 0.0, 1.0, 2.0], device="cuda"), seed=3)
    bias = torch.zeros(8, device="cuda")
    bias[2:5] = 5.0
    y, ids, weights = _call(ops, 3, scoring=scoring, bias=bias, renormalize=False)
    assert torch.equal(ids, torch.tensor([2, 3, 4], device="cuda").expand(3, 3))
    assert bool((weights == 0).all()) and bool((y == 0).all())


@pytest.mark.parametrize("T", [1, 4, 20])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("biased", [False, True])
def test_nan_logit_of_one_expert_under_softmax(T, renormalize, biased):
    """A softmax over a NaN is a NaN everywhere, whichever experts are chosen."""
    ops = list(_layer(T, 8, torch.arange(8.0, device="cuda"), seed=4))
    ops[3][2, 1] = float("nan")  # a NaN in one expert's router row: the least likely choice
    bias = 0.5 * torch.ones(8, device="cuda") if biased else None
    y, ids, weights = _call(ops, 3, renormalize=renormalize, bias=bias)
    assert bool(torch.isnan(weights).all()) and bool(torch.isnan(y).all())
    assert bool(((ids >= 0) & (ids < 8)).all())
    assert all(len(set(row)) == 3 for row in ids.tolist())


@pytest.mark.parametrize("T", [1, 4, 20])
def test_nan_logit_of_one_expert_under_sigmoid(T):
    """Scores of their own: the expert is chosen last, and the others' weights do not know it."""
    ops = list(_layer(T, 8, torch.arange(8.0, device="cuda") - 4, seed=5))
    want = _call(ops, 3, scoring="sigmoid")
    broken = list(ops)
    broken[3] = ops[3].clone()
    broken[3][2, 1] = float("nan")
    for got, ref in zip(_call(broken, 3, scoring="sigmoid"), want):
        assert torch.equal(got, ref)


@pytest.mark.parametrize("T", [1, 4, 20])
def test_logits_of_minus_infinity(T):
    """Masked experts: no weight, and no NaN while any other is left."""
    ops = list(_layer(T, 8, torch.arange(8.0, device="cuda"), seed=6))
    ops[3][4:, 0] = float("-inf")
    y, ids, weights = _call(ops, 3)
    p = torch.softmax(torch.arange(4.0, dtype=torch.float64, device="cuda"), 0).flip(0)[:3]
    assert torch.equal(ids, torch.tensor([3, 2, 1], device="cuda").expand(T, 3))
    assert torch.allclose(weights, (p / p.sum()).expand(T, 3), rtol=1e-4, atol=1e-35)
    assert bool(torch.isfinite(y).all())


@pytest.mark.parametrize("T", [1, 20])
@pytest.mark.parametrize("renormalize", [True, False])
def test_infinite_logit_that_a_bias_passes_over(T, renormalize):
    """inf - inf in the softmax's sum: no weight of the token is a number, whoever is chosen."""
    ops = list(_layer(T, 8, torch.arange(8.0, device="cuda"), seed=7))
    ops[3][7, 0] = float("inf")
    bias = torch.zeros(8, device="cuda")
    bias[:3] = 100.0
    y, ids, weights = _call(ops, 3, renormalize=renormalize, bias=bias)
    assert bool(torch.isnan(weights).all()) and bool(torch.isnan(y).all())


@pytest.mark.parametrize("T,E,k,H,I", [(64, 24, 6, 1024, 128), (40, 60, 4, 512, 128), (16, 8, 4, 2048, 256), (6, 16, 4, 1024, 128)])
def test_scales_of_hidden_rows_that_other_ctas_write(T, E, k, H, I):
    """One or two hidden groups a row: the scales of up to eight rows share a 32-byte piece of memory, and
    each expert's are written by other CTAs just before they are read. Every repeat gives the same bits."""
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    q, s, _, n = tb.rms_norm_fp8(x, torch.ones(H, dtype=torch.bfloat16, device="cuda"), 1e-6, return_normalized=True)
    router = (0.05 * torch.randn(E, H, generator=g, device="cuda")).to(torch.bfloat16)
    w13 = quantize_experts((0.05 * torch.randn(E, 2 * I, H, generator=g, device="cuda")).to(torch.bfloat16))
    w2 = quantize_experts((0.05 * torch.randn(E, H, I, generator=g, device="cuda")).to(torch.bfloat16))
    workspace = tb.moe_workspace(T, E, k, H, I)
    workspace[256:] = 0xFF  # NaN codes and scales from before: a read that comes too early shows
    first = tb.moe_fp8(n, q, s, router, *w13, *w2, top_k=k, workspace=workspace)
    assert bool(torch.isfinite(first).all())
    for _ in range(40):
        workspace[256:] = 0xFF
        assert torch.equal(tb.moe_fp8(n, q, s, router, *w13, *w2, top_k=k, workspace=workspace), first)
