"""The layer of many tokens as a whole (examples/moe_training.py), and its torch.library ops.

Tolerances of the example: e4m3 rounds an element by at most 2^-4, 2^-4 /
sqrt(3) in the mean square; a product of two cast operands carries both
(0.051), the layer's two products with a cast in between at most twice that in
the root of the sum of squares, a gradient through it twice as many factors: 0.15, and
the router's gradient is a difference of the experts' results, whose common
part falls out: twice that. The prefill's hidden rows are rounded to bf16 before
the cast to e4m3, which moves at most 2^-8 / 2^-4 = 1/16 of the codes by a step of
at most 2^-3: 2^-3 / 4 = 0.031 in the mean square, and two roundings of 2^-9 more.
The optimizer's first step is -lr g / (|g| + eps), in fp32.
"""

import importlib.util
from pathlib import Path

import pytest
import torch

import thingy_b200 as tb

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "moe_training.py"
    spec = importlib.util.spec_from_file_location("moe_training", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("tokens", [1, 77, 500])
def test_training_step(example, tokens):
    errors = example.training_step(tokens=tokens)
    assert set(errors) == {"x", "router", "w13", "w2", "step"}
    assert all(0 < errors[k] < 0.15 for k in ("x", "w13", "w2")), errors
    assert 0 < errors["router"] < 0.3, errors
    assert errors["step"] < 1e-3, errors


@pytest.mark.parametrize("tokens", [1, 30, 64])
def test_prefill(example, tokens):
    assert example.prefill(tokens=tokens)["rows"] < 0.035


def test_gradients_captured(example):
    """Forward and backward in a graph, replayed with other tokens. (No eager graph of the leaves may live meanwhile:
    torch then refuses the capture, as for any operator.)"""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = [torch.randn(90, 256, generator=g, device="cuda").bfloat16() for _ in range(2)]
    router = (0.05 * torch.randn(6, 256, generator=g, device="cuda")).bfloat16().requires_grad_()
    w13 = (0.05 * torch.randn(6, 256, 256, generator=g, device="cuda")).requires_grad_()
    w2 = (0.05 * torch.randn(6, 256, 128, generator=g, device="cuda")).requires_grad_()
    place = x[0].clone().requires_grad_()
    leaves = (place, router, w13, w2)

    def step():
        y = example.moe_layer(*leaves, 2)
        return y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y))

    want = []
    for v in x:
        with torch.no_grad():
            place.copy_(v)
        want.append([t.clone() for t in step()])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in (0, 1, 0):
        with torch.no_grad():
            place.copy_(x[i])
        graph.replay()
        for a, b in zip(got, want[i]):
            assert torch.equal(a, b)


def test_another_stream(example):
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(200, 256, generator=g, device="cuda").bfloat16()
    router = (0.05 * torch.randn(6, 256, generator=g, device="cuda")).bfloat16()
    w13 = (0.05 * torch.randn(6, 256, 256, generator=g, device="cuda")).bfloat16()
    w2 = (0.05 * torch.randn(6, 256, 128, generator=g, device="cuda")).bfloat16()
    want = example.moe_layer(x, router, w13, w2, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [example.moe_layer(x, router, w13, w2, 2) for _ in range(3)]
    here = example.moe_layer(x, router, w13, w2, 2)  # both at once
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(t, want) for t in (*got, here))


def test_library_ops():
    import thingy_b200.custom_ops as ops

    g = torch.Generator(device="cuda").manual_seed(0)
    ids = torch.randint(-1, 8, (30, 2), generator=g, device="cuda", dtype=torch.int32)
    x = torch.randn(30, 256, generator=g, device="cuda").bfloat16()
    w = torch.rand(30, 2, generator=g, device="cuda")
    b, sb = tb.quantize_experts((0.05 * torch.randn(8, 128, 256, generator=g, device="cuda")).bfloat16())

    @torch.compile(fullgraph=True, backend="eager")
    def layer(ids, x, w):
        sources, positions, offsets, counts = torch.ops.thingy_b200.moe_sort(ids, 8, 128)
        rows = torch.ops.thingy_b200.moe_permute(x, sources, positions)
        q, s, _, _ = torch.ops.thingy_b200.two_way_cast_to_fp8(rows, False)
        y = torch.ops.thingy_b200.fp8_grouped_gemm(q, s, b, sb, offsets, counts, False)
        return torch.ops.thingy_b200.moe_combine(y, w, sources, positions)

    plan = tb.moe_sort(ids, 8, align=128)
    q, s, _, _ = tb.two_way_cast_to_fp8(tb.moe_permute(x, plan))
    assert torch.equal(layer(ids, x, w), tb.moe_combine(tb.fp8_grouped_gemm(q, s, b, sb, plan), w, plan))
    for op, a in ((ops.moe_sort_op, (ids, 8, 128)), (ops.moe_permute_op, (x, plan.sources, plan.positions)),
                  (ops.moe_combine_op, (x.new_zeros(plan.sources.shape[0], 64), w, plan.sources, plan.positions)),
                  (ops.fp8_grouped_gemm_op, (q, s, b, sb, plan.offsets, plan.counts, True))):
        torch.library.opcheck(op, a, test_utils="test_faketensor")
