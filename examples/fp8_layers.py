"""The 8-bit layers together, as a model uses them: a training step and a decoding step.

    python examples/fp8_layers.py

Training: RMSNorm with its residual, then a gated MLP of three ``fp8_linear``
layers, forward and backward, one weight cast each for the step. Decoding: the
fused RMSNorm -> FP8 kernel makes the rows' codes once; a projection
(``fp8_block_gemm``) reads them, and after the next norm a mixture-of-experts
layer (``moe_fp8``) does, its router the normalized rows. Both print how far
they are from the same layers in 32 bits.
"""

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import thingy_b200 as tb  # noqa: E402

EPS = 1e-6


def relative(got: torch.Tensor, want: torch.Tensor) -> float:
    return ((got.float() - want.float()).norm() / want.float().norm()).item()


def training_step(tokens=300, width=512, hidden=1024, seed=0):
    """Relative errors of the loss's gradients against the layers in 32 bits."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=g, device="cuda")).to(torch.bfloat16).requires_grad_()

    x, residual = normal(tokens, width), normal(tokens, width)
    norm = torch.ones(width, dtype=torch.bfloat16, device="cuda").requires_grad_()
    gate, up, down = normal(hidden, width, scale=0.05), normal(hidden, width, scale=0.05), normal(width, hidden, scale=0.05)
    target = torch.randn(tokens, width, generator=g, device="cuda")
    leaves = (x, residual, norm, gate, up, down)

    def loss(linear, normalized, stream):
        h = torch.nn.functional.silu(linear(normalized, gate)) * linear(normalized, up)
        return (stream.float() + linear(h.to(normalized.dtype), down).float() - target).square().mean()

    _, _, stream, normalized = tb.ResidualRMSNormFP8.apply(x, residual, norm, EPS)
    ours = torch.autograd.grad(loss(tb.fp8_linear, normalized, stream), leaves)
    s32 = x.float() + residual.float()
    n32 = s32 * torch.rsqrt(s32.square().mean(1, keepdim=True) + EPS) * norm.float()
    plain = torch.autograd.grad(loss(lambda a, w: a @ w.float().t(), n32, s32), leaves)
    return {name: relative(a, b) for name, a, b in zip(("x", "residual", "norm", "gate", "up", "down"), ours, plain)}


def decoding_step(tokens=4, width=512, experts=16, hidden=256, top_k=4, seed=0):
    """The step's rows against the same layers in 32 bits on the dequantized weights."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=g, device="cuda")).to(torch.bfloat16)

    x, residual = normal(tokens, width), normal(tokens, width)
    norm1, norm2 = torch.ones_like(x[0]), torch.ones_like(x[0])
    proj, proj_s = tb.per_block_cast_to_fp8(normal(width, width, scale=0.05))
    router = normal(experts, width, scale=0.05)
    w13 = tb.quantize_experts(normal(experts, 2 * hidden, width, scale=0.05))
    w2 = tb.quantize_experts(normal(experts, width, hidden, scale=0.05))

    q, s, stream, _ = tb.rms_norm_fp8(x, norm1, EPS, residual=residual)
    y = tb.fp8_block_gemm(q, s, proj, proj_s)
    q, s, stream, normalized = tb.rms_norm_fp8(y, norm2, EPS, residual=stream, return_normalized=True)
    out = tb.moe_fp8(normalized, q, s, router, *w13, *w2, top_k=top_k)

    def spread(w, scale):
        return w.float() * scale.repeat_interleave(128, -2).repeat_interleave(128, -1)

    def rms(t):
        return t * torch.rsqrt(t.square().mean(1, keepdim=True) + EPS)

    s32 = x.float() + residual.float()
    s32 = s32 + rms(s32) @ spread(proj, proj_s).t()
    n32 = rms(s32)
    p = torch.softmax(normalized.float() @ router.float().t(), 1)
    top = p.topk(top_k, 1)
    weight = torch.zeros_like(p).scatter(1, top.indices, top.values / top.values.sum(1, keepdim=True))
    h = torch.einsum("th,enh->etn", n32, spread(*w13))
    h = torch.nn.functional.silu(h[..., :hidden]) * h[..., hidden:]
    want = torch.einsum("te,eth->th", weight, torch.einsum("eti,ehi->eth", h, spread(*w2)))
    return {"stream": relative(stream, s32), "moe": relative(out, want)}


def main():
    for name, errors in (("training step, gradients", training_step()), ("decoding step", decoding_step())):
        print(f"{name}: " + ", ".join(f"{k} {v:.3f}" for k, v in errors.items()))


if __name__ == "__main__":
    main()
