"""A mixture-of-experts layer with many tokens: a training step with its optimizer, and a prefill.

    python examples/moe_training.py

Training: router, ``moe_sort``, ``moe_permute``, two ``fp8_grouped_linear``
layers with SwiGLU between, ``moe_combine``, backward through all of it, and a
step of ``AdamW`` with 8-bit states on fp32 weights. Prefill: the codes that
``rms_norm_fp8`` made of the tokens go to their experts as they are
(``moe_permute`` of codes and of scales, ``fp8_grouped_gemm``). Both print how far they
are: the gradients from the same layer in 32 bits, the prefill from ``moe_fp8``,
which does the same for up to 64 tokens in one kernel.
"""

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import thingy_b200 as tb  # noqa: E402


def relative(got: torch.Tensor, want: torch.Tensor) -> float:
    return ((got.float() - want.float()).norm() / want.float().norm()).item()


def choose(x, router, top_k):
    """Softmax scores of the chosen experts, renormalized, and their ids."""
    p = torch.softmax(x.float() @ router.float().t(), 1)
    top = p.topk(top_k, 1)
    return top.values / top.values.sum(1, keepdim=True), top.indices


def moe_layer(x, router, w13, w2, top_k):
    """bf16 [T, H]: w13 fp32 or bf16 [E, 2 I, H] (gate rows, then up rows), w2 [E, H, I]."""
    weights, ids = choose(x, router, top_k)
    plan = tb.moe_sort(ids, w13.shape[0], align=128)
    rows = tb.fp8_grouped_linear(tb.moe_permute(x, plan), w13, plan)
    gate, up = rows.chunk(2, 1)
    rows = tb.fp8_grouped_linear(torch.nn.functional.silu(gate) * up, w2, plan)
    return tb.moe_combine(rows, weights, plan)


def moe_layer_32(x, router, w13, w2, top_k):
    """The same in 32 bits, every expert over every token."""
    weights, ids = choose(x, router, top_k)
    spread = torch.zeros(x.shape[0], w13.shape[0], device=x.device).scatter(1, ids, weights)
    gate, up = torch.einsum("th,enh->etn", x.float(), w13.float()).chunk(2, 2)
    rows = torch.einsum("eti,ehi->eth", torch.nn.functional.silu(gate) * up, w2.float())
    return torch.einsum("te,eth->th", spread, rows)


def training_step(tokens=500, width=512, experts=12, hidden=256, top_k=3, seed=0):
    """Relative errors of the gradients, and the optimizer's own distance from the formula."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def leaf(*shape, scale, dtype):
        return (scale * torch.randn(*shape, generator=g, device="cuda")).to(dtype).requires_grad_()

    x = leaf(tokens, width, scale=1.0, dtype=torch.bfloat16)
    router = leaf(experts, width, scale=0.05, dtype=torch.bfloat16)
    w13 = leaf(experts, 2 * hidden, width, scale=0.05, dtype=torch.float32)
    w2 = leaf(experts, width, hidden, scale=0.05, dtype=torch.float32)
    leaves = {"x": x, "router": router, "w13": w13, "w2": w2}
    target = torch.randn(tokens, width, generator=g, device="cuda")

    def loss(layer):
        return (layer(x, router, w13, w2, top_k).float() - target).square().mean()

    plain = torch.autograd.grad(loss(moe_layer_32), list(leaves.values()))
    optimizer = tb.AdamW([router, w13, w2], lr=1e-3, weight_decay=0.0, state_bits=8)
    before = w13.detach().clone()
    loss(moe_layer).backward()
    errors = {name: relative(t.grad, p) for (name, t), p in zip(leaves.items(), plain)}
    norm = torch.stack([t.grad.float().norm() for t in (router, w13, w2)]).norm()
    optimizer.step(grad_scale=(1.0 / norm).clamp(max=1.0).reshape(1))
    # the first step of AdamW is the rate times the gradient's sign, but where eps counts
    clipped = w13.grad * (1.0 / norm).clamp(max=1.0)
    errors["step"] = relative(w13.detach() - before, -1e-3 * clipped / (clipped.abs() + 1e-8))
    return errors


def prefill(tokens=64, width=512, experts=16, hidden=256, top_k=4, seed=0):
    """The layer on codes against the one-kernel layer for few tokens."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=g, device="cuda")).to(torch.bfloat16)

    q, s, _, x = tb.rms_norm_fp8(normal(tokens, width), torch.ones_like(normal(width)), return_normalized=True)
    router = normal(experts, width, scale=0.05)
    w13 = tb.quantize_experts(normal(experts, 2 * hidden, width, scale=0.05))
    w2 = tb.quantize_experts(normal(experts, width, hidden, scale=0.05))
    ids = torch.empty(tokens, top_k, dtype=torch.int32, device="cuda")
    weights = torch.empty(tokens, top_k, device="cuda")
    want = tb.moe_fp8(x, q, s, router, *w13, *w2, top_k=top_k, topk_ids=ids, topk_weights=weights)

    plan = tb.moe_sort(ids, experts, align=128)
    rows = tb.fp8_grouped_gemm(tb.moe_permute(q, plan), tb.moe_permute(s, plan), *w13, plan, out_dtype=torch.float32)
    gate, up = rows.chunk(2, 1)
    h, hs = tb.per_token_cast_to_fp8((torch.nn.functional.silu(gate) * up).bfloat16(), False)
    rows = tb.fp8_grouped_gemm(h, hs, *w2, plan, out_dtype=torch.float32)
    return {"rows": relative(tb.moe_combine(rows, weights, plan), want)}


def main():
    for name, errors in (("training step", training_step()), ("prefill", prefill())):
        print(f"{name}: " + ", ".join(f"{k} {v:.4f}" for k, v in errors.items()))


if __name__ == "__main__":
    main()
