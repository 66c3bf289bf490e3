"""The 8-bit linear-layer operators over their real range: casts, block-scaled products, a training step, a mixture of experts.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits) or, where ``own`` is
true, through this repository's public entry points. ``exact`` computes the same from the definition in 64 bits.

The operators:

* ``cast``: a bf16 matrix to e4m3 codes with fp32 scales, together with the codes of its transpose: weights in
  128 x 128 blocks (one scale a block, both orientations share it), activations and gradients in 1 x 128
  groups along each of the two axes (the products of a training step contract over either).
* ``gemm``: ``D = dequant(A) @ dequant(B).T``, A in 1 x 128 groups, B in 128 x 128 blocks (a layer's product and
  its input gradient) or in 1 x 128 groups too (the weight gradient).
* ``linear``: one training step of a linear layer: casts, the product, the input's and the weight's gradient.
* ``moe``: a whole mixture-of-experts layer for a few tokens: router, top-k, gate and up products, SwiGLU, the
  8-bit cast of the hidden rows, the down product and the weighted sum.
"""

import math

import torch

own = False

F8 = torch.float8_e4m3fn
GROUP = 128
FLOOR = 1e-4  # the least scale: max(amax / 448, 1e-4), the rule of the repository's activation quantizer


def listed():
    return [
        # a large layer's weight after an optimizer step: codes for the product and for the input gradient
        {"name": "cast_weight_8192x8192", "op": "cast", "kind": "block", "rows": 8192, "cols": 8192, "pow2": False},
        # activations of a full training batch, for the product and for the weight gradient
        {"name": "cast_act_16384x7168", "op": "cast", "kind": "both", "rows": 16384, "cols": 7168, "pow2": False},
        # a short ragged batch of gradients with power-of-two scales: the smallest call, launch-bound
        {"name": "cast_grad_77x2056", "op": "cast", "kind": "both", "rows": 77, "cols": 2056, "pow2": True},
        # decoding one token through a square projection: the weight's bytes alone
        {"name": "gemm_decode_1x5120x5120", "op": "gemm", "kind": "block", "M": 1, "N": 5120, "K": 5120, "out": "bf16"},
        # decoding a small batch
        {"name": "gemm_decode_24x7168x5120", "op": "gemm", "kind": "block", "M": 24, "N": 7168, "K": 5120, "out": "bf16"},
        # prefill, or a training batch's forward: the largest product
        {"name": "gemm_prefill_16384x7168x7168", "op": "gemm", "kind": "block", "M": 16384, "N": 7168, "K": 7168, "out": "bf16"},
        # a weight gradient in fp32 over a ragged number of tokens (K is the token axis), scales on both rows
        {"name": "gemm_wgrad_5120x4096x8200", "op": "gemm", "kind": "group", "M": 5120, "N": 4096, "K": 8200, "out": "f32"},
        # one training step of a projection: three casts and three products
        {"name": "linear_step_8192x5120x5120", "op": "linear", "M": 8192, "N": 5120, "K": 5120},
        # the same for a short packed sequence and odd widths
        {"name": "linear_step_1001x1544x2048", "op": "linear", "M": 1001, "N": 1544, "K": 2048},
        # one token through a layer of many experts: the latency of a single request
        {"name": "moe_1_e128_5120x1280", "op": "moe", "T": 1, "E": 128, "k": 8, "H": 5120, "I": 1280, "scoring": "softmax"},
        # a handful of requests, few large experts
        {"name": "moe_7_e8_4096x2048", "op": "moe", "T": 7, "E": 8, "k": 2, "H": 4096, "I": 2048, "scoring": "softmax"},
        # a decoding batch that reaches nearly every expert
        {"name": "moe_64_e64_7168x1024", "op": "moe", "T": 64, "E": 64, "k": 6, "H": 7168, "I": 1024, "scoring": "sigmoid"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["cast", "gemm", "gemm", "linear", "moe", "moe"])
    if op == "cast":
        rows, cols = _log(rng, 1, 16384), 8 * _log(rng, 16, 896)
        return {"op": op, "kind": rng.choice(["block", "both"]), "rows": rows, "cols": cols, "pow2": rng.random() < 0.3}
    if op == "gemm":
        if rng.random() < 0.3:  # weight gradients: the contraction is over any number of tokens
            return {"op": op, "kind": "group", "M": _log(rng, 128, 8192), "N": _log(rng, 128, 8192), "K": _log(rng, 16, 8192),
                    "out": rng.choice(["f32", "f32", "bf16"])}
        return {"op": op, "kind": "block", "M": _log(rng, 1, 16384), "N": 8 * _log(rng, 16, 896), "K": 16 * _log(rng, 8, 448),
                "out": rng.choice(["bf16", "bf16", "f32"])}
    if op == "linear":
        return {"op": op, "M": _log(rng, 32, 8192), "N": 8 * _log(rng, 16, 640), "K": 8 * _log(rng, 16, 640)}
    E = rng.choice([4, 8, 16, 32, 60, 64, 128])
    H = 128 * rng.randint(4, 56)
    I = 128 * rng.randint(1, max(1, min(16, int(4.7e8 / (E * H * 128)))))  # at most the weights of the largest listed case
    return {"op": op, "T": _log(rng, 1, 64), "E": E, "k": rng.randint(1, min(8, E)), "H": H, "I": I,
            "scoring": rng.choice(["softmax", "sigmoid"])}


# ------------------------------------------------------------------ inputs


def _rows(t, n):
    """Each row's scale `n` times along the last axis."""
    return t.repeat_interleave(n, dim=-1)


def _groups(x, dim):
    """The magnitude's maximum over groups of 128 along `dim` (0 or 1) of a matrix; a ragged last group has fewer."""
    x = x.abs()
    if dim == 0:
        x = x.t()
    pad = -x.shape[1] % GROUP
    x = torch.nn.functional.pad(x, (0, pad)).reshape(x.shape[0], -1, GROUP).amax(2)
    return x.t() if dim == 0 else x


def _scale(amax, pow2=False):
    s = (amax / 448.0).clamp_min(FLOOR)
    return torch.exp2(torch.ceil(torch.log2(s))) if pow2 else s


def _quant_rows(x, pow2=False):
    """e4m3 codes and scales of 1 x 128 groups along the rows."""
    s = _scale(_groups(x, 1), pow2)
    return (x / _rows(s, GROUP)[:, : x.shape[1]]).to(F8), s


def _blocks(s, rows, cols):
    """A scale a 128 x 128 block, spread to the elements."""
    return s.repeat_interleave(GROUP, 0)[:rows].repeat_interleave(GROUP, 1)[:, :cols]


def _quant_blocks(w, pow2=False):
    s = _scale(_groups(_groups(w, 1), 0), pow2)
    return (w / _blocks(s, *w.shape)).to(F8), s


def _activations(g, rows, cols):
    """Normalized activations: unit variance, one channel in a hundred fifty times as large."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    big = torch.rand(cols, generator=g, device="cuda") < 0.01
    return torch.where(big, 50.0 * x, x).to(torch.bfloat16)


def _strided(t):
    """Rows on 16-byte boundaries, whatever the width: as the casts lay their codes out."""
    rows, cols = t.shape
    out = torch.zeros(rows, -(-cols // 16) * 16, dtype=t.dtype, device=t.device)
    out[:, :cols] = t
    return out[:, :cols]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] == "cast":
        if case["kind"] == "block":
            state["x"] = (0.02 * torch.randn(case["rows"], case["cols"], generator=g, device="cuda")).to(torch.bfloat16)
        else:
            state["x"] = _activations(g, case["rows"], case["cols"])
    elif case["op"] == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        state["a"], state["sa"] = _quant_rows(_activations(g, M, K).float())
        if case["kind"] == "block":
            state["b"], state["sb"] = _quant_blocks(0.02 * torch.randn(N, K, generator=g, device="cuda"))
        else:
            state["b"], state["sb"] = _quant_rows(1e-3 * _activations(g, N, K).float())
            state["sb"] = state["sb"].t().contiguous().t()  # as the two-way cast lays its scales out
            state["sa"] = state["sa"].t().contiguous().t()
        state["a"], state["b"] = _strided(state["a"]), _strided(state["b"])
    elif case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        state["x"] = _activations(g, M, K)
        state["w"] = (0.02 * torch.randn(N, K, generator=g, device="cuda")).to(torch.bfloat16)
        state["dy"] = (0.1 * torch.randn(M, N, generator=g, device="cuda")).to(torch.bfloat16)
    else:
        T, E, H, I = case["T"], case["E"], case["H"], case["I"]
        x = _activations(g, T, H)
        state["x"] = x
        state["q"], state["s"] = _quant_rows(x.float())
        state["router"] = (0.004 * torch.randn(E, H, generator=g, device="cuda")).to(torch.bfloat16)

        def weight(rows, cols):
            codes = torch.empty(E, rows, cols, dtype=F8, device="cuda")
            for e in range(E):
                codes[e] = (110.0 * torch.randn(rows, cols, generator=g, device="cuda")).clamp(-448, 448).to(F8)
            scale = (0.02 / 110.0) * (0.75 + 0.5 * torch.rand(E, rows // GROUP, cols // GROUP, generator=g, device="cuda"))
            return codes, scale

        state["w13"], state["s13"] = weight(2 * I, H)  # rows 0..I: gate, I..2I: up
        state["w2"], state["s2"] = weight(H, I)
    return state


# ------------------------------------------------------------------ the plain forms


def _plain_cast(x, kind, pow2):
    x = x.float()
    if kind == "block":
        q, s = _quant_blocks(x, pow2)
        return {"q": q, "s": s, "qt": q.t().contiguous(), "st": s.t().contiguous()}
    q, s = _quant_rows(x, pow2)
    qt, st = _quant_rows(x.t().contiguous(), pow2)
    return {"q": q, "s": s, "qt": qt, "st": st}


def _dequant(q, s, kind, dtype=torch.float32):
    spread = _blocks(s, *q.shape) if kind == "block" else _rows(s, GROUP)[:, : q.shape[1]]
    return q.to(dtype) * spread.to(dtype)


def _plain_gemm(a, sa, b, sb, kind):
    return _dequant(a, sa, "group") @ _dequant(b, sb, kind).t()


def _plain_linear(x, w, dy):
    xc, wc, dc = _plain_cast(x, "both", False), _plain_cast(w, "block", False), _plain_cast(dy, "both", False)
    y = _plain_gemm(xc["q"], xc["s"], wc["q"], wc["s"], "block")
    dx = _plain_gemm(dc["q"], dc["s"], wc["qt"], wc["st"], "block")
    dw = _plain_gemm(dc["qt"], dc["st"], xc["qt"], xc["st"], "group")
    return y.to(torch.bfloat16), dx.to(torch.bfloat16), dw.to(torch.bfloat16)


def _plain_moe(s, dtype=torch.float32):
    c = s["case"]
    T, E, k, I = c["T"], c["E"], c["k"], c["I"]
    logits = s["x"].to(dtype) @ s["router"].to(dtype).t()
    if c["scoring"] == "softmax":
        p = torch.exp(logits - logits.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-logits))
    # the scores grow with the logits: chosen by the logits, which do not saturate; ties to the lowest index
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    top = p.gather(1, ids)
    weight = torch.zeros(T, E, dtype=dtype, device=p.device).scatter(1, ids, top / top.sum(1, keepdim=True))

    def spread(w, sw):
        return w.to(dtype) * sw.to(dtype).repeat_interleave(GROUP, 1).repeat_interleave(GROUP, 2)

    act = _dequant(s["q"], s["s"], "group", dtype)
    h = torch.einsum("th,enh->etn", act, spread(s["w13"], s["s13"]))
    gate, up = h[..., :I], h[..., I:]
    h = (gate / (1.0 + torch.exp(-gate)) * up).reshape(E * T, I)
    sh = (_groups(h, 1) / 448.0).clamp_min(FLOOR)
    h = (h / _rows(sh, GROUP)).float().to(F8).to(dtype) * _rows(sh, GROUP)
    y = torch.einsum("eti,ehi->eth", h.reshape(E, T, I), spread(s["w2"], s["s2"]))
    return torch.einsum("te,eth->th", weight, y)


DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def run(state):
    case = state["case"]
    if own:
        return _own(state)
    if case["op"] == "cast":
        return _plain_cast(state["x"], case["kind"], case["pow2"])
    if case["op"] == "gemm":
        return _plain_gemm(state["a"], state["sa"], state["b"], state["sb"], case["kind"]).to(DTYPES[case["out"]])
    if case["op"] == "linear":
        return _plain_linear(state["x"], state["w"], state["dy"])
    return _plain_moe(state).to(torch.bfloat16)


def _own(state):
    import thingy_b200 as tb

    case = state["case"]
    if case["op"] == "cast":
        if case["kind"] == "block":
            q, s, qt, st = tb.per_block_cast_to_fp8(state["x"], case["pow2"], transposed=True)
        else:
            q, s, qt, st = tb.two_way_cast_to_fp8(state["x"], case["pow2"])
        return {"q": q, "s": s, "qt": qt, "st": st}
    if case["op"] == "gemm":
        return tb.fp8_block_gemm(state["a"], state["sa"], state["b"], state["sb"], out_dtype=DTYPES[case["out"]])
    if case["op"] == "linear":
        x, w = state["x"].detach().requires_grad_(), state["w"].detach().requires_grad_()
        y = tb.fp8_linear(x, w)
        dx, dw = torch.autograd.grad(y, (x, w), state["dy"])
        return y, dx, dw
    return tb.moe_fp8(state["x"], state["q"], state["s"], state["router"], state["w13"], state["s13"], state["w2"], state["s2"],
                      top_k=case["k"], scoring=case["scoring"])


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    if case["op"] == "cast":
        n = case["rows"] * case["cols"]
        rb, cb = -(-case["rows"] // GROUP), -(-case["cols"] // GROUP)
        scales = 2 * rb * cb if case["kind"] == "block" else case["rows"] * cb + case["cols"] * rb
        return {"bytes": 2 * n + 2 * n + 4 * scales, "flops": 2 * n}
    if case["op"] == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        kb = -(-K // GROUP)
        sb = -(-N // GROUP) * kb if case["kind"] == "block" else N * kb
        return {"bytes": M * K + N * K + 4 * (M * kb + sb) + M * N * (2 if case["out"] == "bf16" else 4), "flops": 2 * M * N * K}
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": 2 * (M * K + N * K + M * N) + 2 * (M * N + M * K + N * K), "flops": 6 * M * N * K}
    T, E, k, H, I = (case[n] for n in ("T", "E", "k", "H", "I"))
    # every token takes k of E experts: the expected number of experts that some token takes
    active = E * (1.0 - (1.0 - k / E) ** T)
    weights = active * 3 * H * I * (1.0 + 4.0 / GROUP**2)
    return {"bytes": weights + 2 * E * H + T * H * (2 + 1 + 4 / GROUP + 2), "flops": T * k * 6 * H * I + 2 * T * E * H}


# ------------------------------------------------------------------ the definition in 64 bits


def _round8(x):
    return x.float().to(F8).double()


def _exact_quant(x, rows, cols, pow2):
    """Codes and scales of rows x cols tiles, from the definition; double throughout but for the codes' own rounding.

    The scale that the codes are divided by is an fp32 value by definition; the one returned is not rounded."""
    R, C = x.shape
    x = x.double()
    full = torch.zeros(-(-R // rows) * rows, -(-C // cols) * cols, dtype=torch.float64, device=x.device)
    full[:R, :C] = x
    amax = full.view(full.shape[0] // rows, rows, full.shape[1] // cols, cols).abs().permute(0, 2, 1, 3).flatten(2).max(2).values
    s = torch.maximum(amax / 448.0, torch.full_like(amax, FLOOR))
    if pow2:
        m, e = torch.frexp(s)  # s = m 2^e, m in [1/2, 1)
        s = torch.ldexp(torch.ones_like(s), torch.where(m == 0.5, e - 1, e))
    spread = s.float().double()[:, None, :, None].expand(-1, rows, -1, cols).reshape(full.shape)[:R, :C]
    return _round8(x / spread), s


def _exact_cast(x, kind, pow2):
    if kind == "block":
        q, s = _exact_quant(x, GROUP, GROUP, pow2)
        return {"q": q, "s": s, "qt": q.t().contiguous(), "st": s.t().contiguous()}
    (q, s), (qt, st) = _exact_quant(x, 1, GROUP, pow2), _exact_quant(x.t(), 1, GROUP, pow2)
    return {"q": q, "s": s, "qt": qt, "st": st}


def _exact_product(a, sa, b, sb):
    """Block by block of the contraction, the scales applied to each block's partial product."""
    K, N = a.shape[1], b.shape[0]
    out = torch.zeros(a.shape[0], N, dtype=torch.float64, device=a.device)
    rows = torch.arange(N, device=a.device) // (GROUP if sb.shape[0] != N else 1)
    for i, k in enumerate(range(0, K, GROUP)):
        part = a[:, k : k + GROUP].double() @ b[:, k : k + GROUP].double().t()
        out += part * sa[:, i : i + 1].double() * sb[rows, i].double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "cast":
        return _exact_cast(s["x"], case["kind"], case["pow2"])
    if case["op"] == "gemm":
        return _exact_product(s["a"], s["sa"], s["b"], s["sb"])
    if case["op"] == "linear":
        x, w, d = _exact_cast(s["x"], "both", False), _exact_cast(s["w"], "block", False), _exact_cast(s["dy"], "both", False)
        return (_exact_product(x["q"], x["s"], w["q"], w["s"]), _exact_product(d["q"], d["s"], w["qt"], w["st"]),
                _exact_product(d["qt"], d["st"], x["qt"], x["st"]))
    T, E, k, H, I = (case[n] for n in ("T", "E", "k", "H", "I"))
    logits = s["x"].double() @ s["router"].double().t()
    p = torch.softmax(logits, 1) if case["scoring"] == "softmax" else torch.sigmoid(logits)
    top = logits.topk(k, dim=1).indices
    weight = p.gather(1, top)
    weight = weight / weight.sum(1, keepdim=True)
    y = torch.zeros(T, H, dtype=torch.float64, device=logits.device)
    for e in range(E):  # only the tokens that take expert e
        t, slot = (top == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        gu = _exact_product(s["q"][t], s["s"][t], s["w13"][e], s["s13"][e])
        h = torch.nn.functional.silu(gu[:, :I]) * gu[:, I:]
        q, sh = _exact_quant(h, 1, GROUP, False)
        y[t] += weight[t, slot, None] * _exact_product(q, sh, s["w2"][e], s["s2"][e])
    return y
