"""The 8-bit layers used together (examples/fp8_layers.py), and as torch.library ops.

Tolerances of the example: e4m3 has 3 mantissa bits, a relative rounding error
of at most 2^-4 an element, 2^-4 / sqrt(3) in the mean square where values
fill a binade evenly. A product of two cast operands carries both (sqrt(2)
2^-4 / sqrt(3) = 0.051), the chain of three products of the MLP at most three
times that in the root of the sum of squares (0.09), a gradient through it
twice as many factors (0.13): below 0.2 everywhere.
"""

import importlib.util
from pathlib import Path

import pytest
import torch

import thingy_b200 as tb

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "fp8_layers.py"
    spec = importlib.util.spec_from_file_location("fp8_layers", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_training_step(example):
    errors = example.training_step()
    assert set(errors) == {"x", "residual", "norm", "gate", "up", "down"}
    assert all(0 < e < 0.2 for e in errors.values()), errors


def test_decoding_step(example):
    errors = example.decoding_step()
    assert errors["stream"] < 0.1 and errors["moe"] < 0.2, errors


def test_library_ops_inside_a_compiled_region():
    import thingy_b200.custom_ops  # noqa: F401

    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(40, 264, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn(136, 264, generator=g, device="cuda").to(torch.bfloat16)

    @torch.compile(fullgraph=True, backend="eager")
    def layer(x, w):
        q, s, qt, st = torch.ops.thingy_b200.two_way_cast_to_fp8(x, False)
        wq, ws, wqt, wst = torch.ops.thingy_b200.per_block_cast_to_fp8(w, False)
        y = torch.ops.thingy_b200.fp8_block_gemm(q, s, wq, ws, False)
        gram = torch.ops.thingy_b200.fp8_block_gemm(qt, st, qt, st, True)
        return y, gram, wqt, wst

    y, gram, wqt, wst = layer(x, w)
    q, s, qt, st = tb.two_way_cast_to_fp8(x)
    wq, ws, wqt2, wst2 = tb.per_block_cast_to_fp8(w, transposed=True)
    assert torch.equal(y, tb.fp8_block_gemm(q, s, wq, ws))
    assert torch.equal(gram, tb.fp8_block_gemm(qt, st, qt, st, out_dtype=torch.float32))
    assert torch.equal(wqt.float(), wqt2.float()) and torch.equal(wst, wst2)


def test_library_op_shapes_match_the_results():
    import thingy_b200.custom_ops as ops

    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(20, 384, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.ones(384, dtype=torch.bfloat16, device="cuda")
    q, s, _, n = tb.rms_norm_fp8(x, w, return_normalized=True)
    router = torch.randn(8, 384, generator=g, device="cuda").to(torch.bfloat16)
    w13 = tb.quantize_experts(torch.randn(8, 512, 384, generator=g, device="cuda").to(torch.bfloat16))
    w2 = tb.quantize_experts(torch.randn(8, 384, 256, generator=g, device="cuda").to(torch.bfloat16))
    args = (n, q, s, router, *w13, *w2, 2, "sigmoid", True, 1.0, None)
    for op, a in ((ops.two_way_cast_op, (x[:, :200], True)), (ops.per_block_cast_op, (x, False)),
                  (ops.fp8_block_gemm_op, (q, s, w13[0][0], w13[1][0], True)), (ops.moe_fp8_op, args)):
        torch.library.opcheck(op, a, test_utils="test_faketensor")  # its schema test lacks float8 arithmetic
