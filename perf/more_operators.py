"""Training and prefill of a mixture of experts in 8 bits: tokens sorted by expert and back, the experts' products, AdamW.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits) or, where ``own`` is
true, through this repository's public entry points. ``exact`` computes the same from the definition in 64 bits.

The operators:

* ``sort``: the choices of T tokens (k experts each) in the order of their experts, stable, every expert's rows
  padded to a multiple of ``align``. Ids below zero are choices that are not made here (dropped, or another rank's).
* ``permute``: the tokens' rows in that order, and the gradient that comes back; or 8-bit codes and their scales.
* ``combine``: the experts' rows back to their tokens, weighted and summed; in training with both gradients.
* ``grouped``: a training step of the experts' linear layer on sorted rows, in 8 bits.
* ``product``: the experts' product alone, on codes that the serving path has.
* ``adamw``: an optimizer step over many tensors, states in 32 bits or in e4m3 codes of groups of 128.
"""

import math

import torch

own = False

F8 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GROUP = 128
FLOOR = 1e-4  # the least scale of weights and activations: max(amax / 448, 1e-4), the repository's rule
LEAST = 2.0**-92  # the least scale of gradients and of optimizer states
MASK = 0xFFFFFFFF


def listed():
    return [
        # one token that is being decoded: latency alone
        {"name": "sort_1x8_e128", "op": "sort", "T": 1, "k": 8, "E": 128, "align": 128, "drop": 0.0},
        # a large training batch over many experts, of which a share is another rank's
        {"name": "sort_32768x8_e256", "op": "sort", "T": 32768, "k": 8, "E": 256, "align": 128, "drop": 0.1},
        # training: a full batch's rows to their experts, and the gradient back
        {"name": "permute_16384x4096_k8", "op": "permute", "T": 16384, "k": 8, "E": 64, "align": 128, "drop": 0.0, "H": 4096, "dtype": "bf16"},
        # prefill of a short prompt: codes and scales
        {"name": "permute_codes_203x7168_k8", "op": "permute", "T": 203, "k": 8, "E": 64, "align": 128, "drop": 0.0, "H": 7168, "dtype": "e4m3"},
        # training: the experts' rows back, and the gradients of rows and weights
        {"name": "combine_8192x5120_k8", "op": "combine", "T": 8192, "k": 8, "E": 64, "align": 128, "drop": 0.0, "H": 5120, "dtype": "bf16", "train": True},
        # a few tokens of an odd width, some choices absent: the smallest
        {"name": "combine_33x1030_k4", "op": "combine", "T": 33, "k": 4, "E": 16, "align": 1, "drop": 0.2, "H": 1030, "dtype": "f16", "train": False},
        # a training step of the experts' projection
        {"name": "grouped_4096x4_e16_2048x4096", "op": "grouped", "T": 4096, "k": 4, "E": 16, "drop": 0.0, "N": 2048, "K": 4096, "weight": "bf16"},
        # the same for a short packed batch over small experts, master weights in fp32
        {"name": "grouped_333x4_e8_640x1024", "op": "grouped", "T": 333, "k": 4, "E": 8, "drop": 0.1, "N": 640, "K": 1024, "weight": "f32"},
        # a prompt's prefill: many rows an expert
        {"name": "product_4096x8_e32_4096x2048", "op": "product", "T": 4096, "k": 8, "E": 32, "drop": 0.0, "N": 4096, "K": 2048, "out": "bf16"},
        # a decoding batch just above what the one-kernel layer takes: every expert's weight once
        {"name": "product_100x6_e64_2048x7168", "op": "product", "T": 100, "k": 6, "E": 64, "drop": 0.0, "N": 2048, "K": 7168, "out": "bf16"},
        # the experts' and the dense weights of a few layers, bf16 with 8-bit states
        {"name": "adamw_8bit_bf16_134M", "op": "adamw", "param": "bf16", "grad": "bf16", "bits": 8, "count": 24, "total": 134217728, "odd": False, "decay": 0.1},
        # master weights in fp32 with all the small tensors of a model: norms, biases, scalars
        {"name": "adamw_32bit_f32_200_tensors", "op": "adamw", "param": "f32", "grad": "f32", "bits": 32, "count": 200, "total": 20000000, "odd": True, "decay": 0.01},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sort", "permute", "combine", "grouped", "product", "adamw"])
    drop = rng.choice([0.0, 0.0, 0.2])
    E = rng.choice([4, 8, 16, 60, 64, 128])
    k = rng.randint(1, min(8, E))
    if op == "sort":
        E = rng.choice([1, 8, 60, 128, 256, 512])
        return {"op": op, "T": _log(rng, 1, 32768), "k": rng.randint(1, min(8, E)), "E": E, "align": rng.choice([1, 16, 128]), "drop": drop}
    if op in ("permute", "combine"):
        H = rng.choice([rng.randint(64, 7168), 8 * rng.randint(16, 896), 128 * rng.randint(1, 56)])
        T = _log(rng, 1, max(1, min(16384, int(5e8 / (H * k)))))
        case = {"op": op, "T": T, "k": k, "E": E, "align": rng.choice([1, 128]), "drop": drop, "H": H}
        if op == "permute":
            return {**case, "dtype": "e4m3" if H % 128 == 0 and rng.random() < 0.5 else rng.choice(["bf16", "bf16", "f16", "f32"])}
        return {**case, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "train": rng.random() < 0.6}
    if op in ("grouped", "product"):
        E = rng.choice([1, 4, 8, 16, 32, 64])
        k = rng.randint(1, min(6, E))
        N, K = 128 * rng.randint(1, 32), 128 * rng.randint(1, 32)
        while E * N * K > 2.5e8:
            E //= 2
        k = min(k, E)
        most = int((1.3e11 if op == "grouped" else 2.6e11) / (N * K * k))
        case = {"op": op, "T": _log(rng, 1, max(1, min(8192, most))), "k": k, "E": E, "drop": drop, "N": N, "K": K}
        return {**case, "weight": rng.choice(["bf16", "f32"])} if op == "grouped" else {**case, "out": rng.choice(["bf16", "bf16", "f32"])}
    param = rng.choice(["bf16", "f32", "f32", "f16"])
    return {"op": op, "param": param, "grad": rng.choice([param, "f32"]), "bits": rng.choice([8, 32]), "count": _log(rng, 1, 400),
            "total": _log(rng, 1000, 60000000), "odd": rng.random() < 0.5, "decay": rng.choice([0.0, 0.1])}


# ------------------------------------------------------------------ inputs


def _ceil(a, b):
    return -(-a // b) * b


def plan_rows(T, k, E, align):
    """The rows that sorted choices can need: every expert that may have some rounds up."""
    n = T * k
    return (n + min(E, n) * (align - 1)) // align * align


def _choices(g, c):
    """k different experts a token; some experts are liked more. A dropped choice is -1."""
    liked = 0.7 * torch.randn(c["E"], generator=g, device="cuda")
    logits = torch.randn(c["T"], c["E"], generator=g, device="cuda") + liked
    ids = torch.topk(logits, c["k"], dim=1).indices.int()
    gone = torch.rand(c["T"], c["k"], generator=g, device="cuda") < c["drop"]
    return torch.where(gone, torch.full_like(ids, -1), ids)


def _sort(ids, E, align):
    """The plan: sources [R], positions [T, k], offsets [E + 1], counts [E], all int32."""
    T, k = ids.shape
    n, R = T * k, plan_rows(T, k, E, align)
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < E), flat, torch.full_like(flat, E))
    order = torch.sort(key, stable=True).indices
    key = key[order]
    counts = torch.zeros(E + 1, dtype=torch.long, device=ids.device).scatter_add_(0, key, torch.ones_like(key))
    first = torch.cumsum(counts, 0) - counts  # in the order without padding
    padded = (counts[:E] + align - 1) // align * align
    offsets = torch.cat([torch.zeros_like(counts[:1]), torch.cumsum(padded, 0)])
    at = offsets[key] + torch.arange(n, device=ids.device) - first[key]
    at = torch.where(key < E, at, torch.full_like(at, -1))
    sources = torch.full((R + 1,), -1, dtype=torch.int32, device=ids.device)
    sources[torch.where(at >= 0, at, torch.full_like(at, R))] = order.int()  # absent choices to a row that is cut off
    positions = torch.zeros(n, dtype=torch.int32, device=ids.device)
    positions[order] = at.int()
    return {"sources": sources[:R].contiguous(), "positions": positions.reshape(T, k), "offsets": offsets.int(), "counts": counts[:E].int()}


def _over(amax):
    """amax / 448, rounded once: a tensor over a number would be a product with the number's rounded reciprocal."""
    return amax / torch.full_like(amax, 448.0)


def _groups(x, dim):
    x = x.abs()
    if dim == 0:
        x = x.t()
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % GROUP)).reshape(x.shape[0], -1, GROUP).amax(2)
    return x.t() if dim == 0 else x


def _scale(amax, gradient=False):
    s = _over(amax)
    if gradient:
        return torch.where(amax < FLOOR, s.clamp_min(LEAST), s.clamp_min(FLOOR))
    return s.clamp_min(FLOOR)


def _spread(s, cols):
    return s.repeat_interleave(GROUP, -1)[..., :cols]


def _quant_rows(x, gradient=False):
    s = _scale(_groups(x, 1), gradient)
    return (x / _spread(s, x.shape[1])).to(F8), s


def _activations(g, rows, cols):
    """Normalized activations: unit variance, one channel in a hundred twenty times as large."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    big = torch.rand(cols, generator=g, device="cuda") < 0.01
    return torch.where(big, 20.0 * x, x).to(torch.bfloat16)


def _gathered(x, plan, k):
    """Rows in sorted order, zeros in padding."""
    src = plan["sources"].long()
    rows = x[src.clamp_min(0) // k]
    return torch.where((src >= 0)[:, None], rows, torch.zeros_like(rows))


def _shapes(c):
    """The tensors' sizes of a model: a few large ones, many small ones, some that are one element."""
    n, total, count = [], c["total"], c["count"]
    for i in range(count):
        if i == count - 1:
            size = max(1, total - sum(n))
        elif c["odd"] and i % 7 == 3:
            size = 1 + i % 3
        else:
            size = max(1, int(total / count * (0.25 + 1.5 * ((i * 37) % 101) / 101)))
            size = size | 1 if c["odd"] and i % 2 else _ceil(size, 64)
        n.append(size)
    return n


def _begins(sizes, odd):
    """Where they begin in a buffer: on 64 elements, but some behind the one before where odd ones are wanted."""
    begin, at = [], 0
    for i, n in enumerate(sizes):
        at = at if odd and i % 5 == 4 else _ceil(at, 64)
        begin.append(at)
        at += n
    return begin


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": c}
    op = c["op"]

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if op == "sort":
        state["ids"] = _choices(g, c)
    elif op in ("permute", "combine"):
        plan = state["plan"] = _sort(_choices(g, c), c["E"], c["align"])
        R, T, k, H = len(plan["sources"]), c["T"], c["k"], c["H"]
        if op == "permute" and c["dtype"] == "e4m3":
            state["x"], state["s"] = _quant_rows(_activations(g, T, H).float())
        elif op == "permute":
            state["x"] = _activations(g, T, H).to(DTYPES[c["dtype"]])
            state["dxs"] = (0.1 * rand(R, H)).to(DTYPES[c["dtype"]])
        else:
            state["ys"] = rand(R, H).to(DTYPES[c["dtype"]])
            w = torch.rand(T, k, generator=g, device="cuda") + 0.05
            state["w"] = w / w.sum(1, keepdim=True)
            state["dy"] = (0.1 * rand(T, H)).to(DTYPES[c["dtype"]])
    elif op in ("grouped", "product"):
        plan = state["plan"] = _sort(_choices(g, c), c["E"], GROUP)
        T, k, E, N, K = c["T"], c["k"], c["E"], c["N"], c["K"]
        x = _gathered(_activations(g, T, K), plan, k)
        if op == "grouped":
            state["x"] = x
            state["w"] = (0.02 * rand(E, N, K)).to(DTYPES[c["weight"]])
            state["dy"] = _gathered((0.1 * rand(T * k, N)).to(torch.bfloat16), plan, 1)
        else:
            state["a"], state["sa"] = _quant_rows(x.float())
            state["b"] = (110.0 * torch.randn(E, N, K, generator=g, device="cuda")).clamp_(-448, 448).to(F8)
            state["sb"] = (0.02 / 110.0) * (0.75 + 0.5 * torch.rand(E, N // GROUP, K // GROUP, generator=g, device="cuda"))
    else:
        # tensors that are views into one buffer each, as a program keeps what it also gathers or stores as a whole
        sizes = _shapes(c)
        begin = _begins(sizes, c["odd"])
        state["at"] = at = list(zip(begin, sizes))
        end = begin[-1] + sizes[-1]
        size = torch.zeros(end, device="cuda")  # of the gradients, another in each tensor
        for a, n in at:
            size[a : a + n] = 1e-3 * torch.exp(2.0 * rand(1))
        grad = (size * rand(end)).to(DTYPES[c["grad"]])
        state["buffers"] = buffers = {"p": (0.02 * rand(end)).to(DTYPES[c["param"]])}
        # the states that some steps of such gradients leave
        m = 0.3 * grad.float() * torch.rand(end, generator=g, device="cuda")
        v = grad.float() ** 2 * (0.2 + torch.rand(end, generator=g, device="cuda"))
        parts = lambda x: [x[a : a + n] for a, n in at]  # noqa: E731
        state["p"], state["g"] = parts(buffers["p"]), parts(grad)
        if c["bits"] == 32:
            buffers["m"], buffers["v"] = m, v
            state["m"], state["v"] = parts(m), parts(v)
        else:
            groups = [_ceil(n, GROUP) // GROUP for n in sizes]
            first = [sum(groups[:i]) for i in range(len(groups))]
            for name, x in (("m", m), ("v", v.sqrt())):
                codes, scales = torch.zeros(end, dtype=F8, device="cuda"), torch.zeros(sum(groups), device="cuda")
                state[name] = [(codes[a : a + n], scales[f : f + k]) for (a, n), f, k in zip(at, first, groups)]
                for (a, n), (q, sc) in zip(at, state[name]):
                    for place, value in zip((q, sc), _state8(x[a : a + n])):
                        place.copy_(value)
                buffers[name], buffers[name + "s"] = codes, scales
        state["step"] = 10
        state["seed"] = seed
        state["lr"] = 1e-3
        state["clip"] = torch.full((1,), 0.7, device="cuda")  # what a clipped norm leaves of the gradients
    return state


def _state8(x):
    """Codes [n] and scales [ceil(n / 128)] of a state, to the nearest."""
    n = x.numel()
    s = _over(torch.nn.functional.pad(x, (0, -n % GROUP)).reshape(-1, GROUP).abs().amax(1)).clamp_min(LEAST)
    return [(x / _spread(s, n)).to(F8), s]


# ------------------------------------------------------------------ the plain forms


def _plain_combine(ys, w, plan):
    pos = plan["positions"].long()
    here = (pos >= 0)[..., None]
    rows = torch.where(here, ys.float()[pos.clamp_min(0)], torch.zeros((), device=ys.device))
    return (w[..., None] * rows).sum(1), rows


def _plain_permute(s):
    c, plan, k = s["case"], s["plan"], s["case"]["k"]
    if c["dtype"] == "e4m3":
        codes = _gathered(s["x"].view(torch.uint8), plan, k).view(F8)
        return {"q": codes, "s": _gathered(s["s"], plan, k)}
    pos = plan["positions"].long()
    rows = torch.where((pos >= 0)[..., None], s["dxs"].float()[pos.clamp_min(0)], torch.zeros((), device=pos.device))
    return {"xs": _gathered(s["x"], plan, k), "dx": rows.sum(1).to(s["x"].dtype)}


def _plain_combine_step(s):
    c, plan, ys, w = s["case"], s["plan"], s["ys"], s["w"]
    y, rows = _plain_combine(ys, w, plan)
    y = y.to(ys.dtype)
    if not c["train"]:
        return {"y": y}
    dy, k = s["dy"].float(), c["k"]
    src = plan["sources"].long()
    dys = dy[src.clamp_min(0) // k] * torch.where(src >= 0, w.reshape(-1)[src.clamp_min(0)], torch.zeros((), device=w.device))[:, None]
    return {"y": y, "dys": dys.to(ys.dtype), "dw": (rows * dy[:, None, :]).sum(2)}


def _dequant_rows(q, s):
    return q.float() * _spread(s, q.shape[1])


def _cast_blocks(w):
    """Weights [E, N, K] on e4m3 codes in 128 x 128 blocks, as the values that they stand for."""
    E, N, K = w.shape
    amax = w.abs().reshape(E, N // GROUP, GROUP, K // GROUP, GROUP).amax((2, 4))
    s = _scale(amax).repeat_interleave(GROUP, 1).repeat_interleave(GROUP, 2)
    return (w / s).to(F8).float() * s


def _tiles(plan, E):
    """The expert of each tile of 128 rows, E for those behind the last."""
    at = GROUP * torch.arange(len(plan["sources"]) // GROUP, device=plan["offsets"].device)
    return torch.searchsorted(plan["offsets"].long()[1:].contiguous(), at, right=True)


def _by_tile(a, w, tiles):
    """Each tile of 128 rows of a times its expert's matrix [K, N], zeros behind the last."""
    E = w.shape[0]
    out = torch.bmm(a.reshape(-1, GROUP, a.shape[1]), w[tiles.clamp_max(E - 1)])
    out = torch.where((tiles < E)[:, None, None], out, torch.zeros((), device=a.device))
    return out.reshape(-1, w.shape[2])


def _plain_grouped(s):
    plan, E = s["plan"], s["case"]["E"]
    tiles = _tiles(plan, E)
    x, dy = s["x"].float(), s["dy"].float()
    w = _cast_blocks(s["w"].to(torch.bfloat16).float())
    y = _by_tile(_dequant_rows(*_quant_rows(x)), w.transpose(1, 2), tiles)
    dx = _by_tile(_dequant_rows(*_quant_rows(dy, True)), w, tiles)
    xt = _dequant_rows(*_quant_rows(x.t())).reshape(x.shape[1], -1, GROUP)
    dt = _dequant_rows(*_quant_rows(dy.t(), True)).reshape(dy.shape[1], -1, GROUP)
    parts = torch.bmm(dt.permute(1, 0, 2), xt.permute(1, 2, 0))  # [tiles, N, K]
    dw = torch.zeros(E + 1, *parts.shape[1:], device=x.device).index_add_(0, tiles, parts)[:E]
    return {"y": y.to(torch.bfloat16), "dx": dx.to(torch.bfloat16), "dw": dw.to(s["w"].dtype)}


def _plain_product(s):
    sb = s["sb"].repeat_interleave(GROUP, 1).repeat_interleave(GROUP, 2)
    w = s["b"].float() * sb
    return _by_tile(_dequant_rows(s["a"], s["sa"]), w.transpose(1, 2), _tiles(s["plan"], s["case"]["E"])).to(DTYPES[s["case"]["out"]])


def _mix(x):
    """A hash of 32 bits: xor-shifts and products with the leading bits of the golden ratio and of the root of two."""
    x = x ^ (x >> 16)
    x = (x * 0x9E3779B9) & MASK
    x = x ^ (x >> 15)
    x = (x * 0x6A09E667) & MASK
    return x ^ (x >> 16)


def _random(n, ordinal, step, seed, device):
    """32 bits for each element of the ordinal-th tensor in a step."""
    key = _mix((seed & MASK) ^ _mix((seed >> 32) & MASK))
    key = _mix(_mix(key ^ (step & MASK)) ^ ordinal)
    return _mix((torch.arange(n, device=device) * 0x9E3779B9 + key) & MASK)


def _round8(y, bits):
    """Magnitudes to e4m3: one of the two neighbours, the nearer one the likelier; bits: 16 random ones an element."""
    small = y < 2.0**-6
    z = torch.where(small, y + 2.0**-6, y)  # subnormals have the spacing of the first binade
    z = ((z.view(torch.int32) + (bits << 4).int()) & -0x100000).view(torch.float32)
    return torch.where(small, z - 2.0**-6, z).clamp_max(448.0)


def _store8(x, bits, positive):
    n = x.numel()
    s = _over(torch.nn.functional.pad(x, (0, -n % GROUP)).reshape(-1, GROUP).abs().amax(1)).clamp_min(LEAST)
    z = _round8(x.abs() * _spread(1.0 / s, n), bits)
    z = torch.where(x > 0, z.clamp_min(2.0**-9), z) if positive else torch.copysign(z, x)
    return z.to(F8), s


def _adamw_one(i, s, step):
    """The i-th tensor: new values into its place."""
    c, lr, b1, b2, eps = s["case"], s["lr"], 0.9, 0.95, 1e-8
    p, g, m, v = s["p"][i], s["g"][i].float() * s["clip"], s["m"][i], s["v"][i]
    n = p.numel()
    if c["bits"] == 8:
        m32 = m[0].float() * _spread(m[1], n)
        r = v[0].float() * _spread(v[1], n)
        v32 = r * r
    else:
        m32, v32 = m, v
    m32 = b1 * m32 + (1.0 - b1) * g
    v32 = b2 * v32 + (1.0 - b2) * (g * g)
    root = torch.sqrt(v32)
    new = p.float() * (1.0 - lr * c["decay"]) - (lr / (1.0 - b1**step)) * (m32 / (root * (1.0 - b2**step) ** -0.5 + eps))
    p.copy_(new)
    if c["bits"] == 8:
        bits = _random(n, i, step, s["seed"], p.device)
        codes, scales = _store8(m32, bits & 0xFFFF, False)
        m[0].copy_(codes)
        m[1].copy_(scales)
        codes, scales = _store8(root, bits >> 16, True)
        v[0].copy_(codes)
        v[1].copy_(scales)
    else:
        m.copy_(m32)
        v.copy_(v32)


def _plain_adamw(s):
    s["step"] += 1
    _ = [_adamw_one(i, s, s["step"]) for i in range(s["case"]["count"])]
    return s["buffers"]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "sort":
        return _sort(state["ids"], state["case"]["E"], state["case"]["align"])
    if op == "permute":
        return _plain_permute(state)
    if op == "combine":
        return _plain_combine_step(state)
    if op == "grouped":
        return _plain_grouped(state)
    return _plain_product(state) if op == "product" else _plain_adamw(state)


def _own(state):
    import thingy_b200 as tb

    c, op = state["case"], state["case"]["op"]
    if op == "sort":
        plan = tb.moe_sort(state["ids"], c["E"], align=c["align"])
        return {"sources": plan.sources, "positions": plan.positions, "offsets": plan.offsets, "counts": plan.counts}
    if op == "adamw":
        state["step"] += 1
        tb.adamw_step(state["p"], state["g"], state["m"], state["v"], step=state["step"], lr=state["lr"], betas=(0.9, 0.95), eps=1e-8,
                      weight_decay=c["decay"], grad_scale=state["clip"], seed=state["seed"])
        return state["buffers"]
    align = c["align"] if "align" in c else GROUP
    plan = tb.MoePlan(state["plan"]["sources"], state["plan"]["positions"], state["plan"]["offsets"], state["plan"]["counts"], align)
    if op == "permute":
        if c["dtype"] == "e4m3":
            return {"q": tb.moe_permute(state["x"], plan), "s": tb.moe_permute(state["s"], plan)}
        x = state["x"].detach().requires_grad_()
        xs = tb.moe_permute(x, plan)
        return {"xs": xs.detach(), "dx": torch.autograd.grad(xs, x, state["dxs"])[0]}
    if op == "combine":
        if not c["train"]:
            return {"y": tb.moe_combine(state["ys"], state["w"], plan)}
        ys, w = state["ys"].detach().requires_grad_(), state["w"].detach().requires_grad_()
        y = tb.moe_combine(ys, w, plan)
        dys, dw = torch.autograd.grad(y, (ys, w), state["dy"])
        return {"y": y.detach(), "dys": dys, "dw": dw}
    if op == "product":
        return tb.fp8_grouped_gemm(state["a"], state["sa"], state["b"], state["sb"], plan, out_dtype=DTYPES[c["out"]])
    x, w = state["x"].detach().requires_grad_(), state["w"].detach().requires_grad_()
    y = tb.fp8_grouped_linear(x, w, plan)
    dx, dw = torch.autograd.grad(y, (x, w), state["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw}


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    c, op = case, case["op"]
    if op == "adamw":
        size = {"bf16": 2, "f16": 2, "f32": 4}
        states = 16 if c["bits"] == 32 else 4 + 16 / GROUP
        return {"bytes": c["total"] * (2 * size[c["param"]] + size[c["grad"]] + states), "flops": 15 * c["total"]}
    T, k, E = c["T"], c["k"], c["E"]
    n = T * k * (1 - c["drop"])  # choices that are made
    R = plan_rows(T, k, E, c.get("align", GROUP))
    if op == "sort":
        return {"bytes": 8 * T * k + 4 * R + 8 * E, "flops": T * k}
    if op == "permute" and c["dtype"] == "e4m3":
        row = c["H"] * (1 + 4 / GROUP)
        return {"bytes": (T + R) * row, "flops": 0}
    if op in ("permute", "combine"):
        row = c["H"] * {"bf16": 2, "f16": 2, "f32": 4}[c["dtype"]]
        if op == "permute":
            return {"bytes": (2 * T + n + R) * row, "flops": n * c["H"]}
        if not c["train"]:
            return {"bytes": (n + T) * row + 8 * T * k, "flops": 2 * n * c["H"]}
        return {"bytes": (2 * n + 2 * T + R) * row + 20 * T * k, "flops": 5 * n * c["H"]}
    N, K = c["N"], c["K"]
    some = E * (1.0 - (1.0 - k / E) ** T)  # experts that some token takes
    if op == "product":
        return {"bytes": some * N * K + n * K * (1 + 4 / GROUP) + n * N * (2 if c["out"] == "bf16" else 4), "flops": 2 * n * N * K}
    w = 2 if c["weight"] == "bf16" else 4
    return {"bytes": 2 * E * N * K * w + 4 * n * (N + K), "flops": 6 * n * N * K}


# ------------------------------------------------------------------ the definition in 64 bits


def _exact_quant(x, rows, cols, gradient=False):
    """What rows x cols tiles of x stand for on e4m3 codes; the scale that codes are divided by is an fp32 value."""
    R, C = x.shape
    t = x.double().reshape(R // rows, rows, C // cols, cols)
    amax = t.abs().amax((1, 3), keepdim=True)
    s = amax / 448.0
    s = torch.where((amax < FLOOR) & torch.tensor(gradient, device=x.device), s.clamp_min(LEAST), s.clamp_min(FLOOR))
    return ((t / s.float().double()).float().to(F8).double() * s).reshape(R, C)


def _exact_sort(ids, E, align):
    T, k = ids.shape
    flat = ids.reshape(-1).cpu().tolist()
    R = plan_rows(T, k, E, align)
    own_rows = [[] for _ in range(E)]
    for i, e in enumerate(flat):
        if 0 <= e < E:
            own_rows[e].append(i)
    sources, positions, offsets = [-1] * R, [-1] * (T * k), [0]
    for rows in own_rows:
        for j, i in enumerate(rows):
            sources[offsets[-1] + j] = i
            positions[i] = offsets[-1] + j
        offsets.append(offsets[-1] + _ceil(len(rows), align))
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device=ids.device)  # noqa: E731
    return {"sources": as_int(sources), "positions": as_int(positions).reshape(T, k), "offsets": as_int(offsets),
            "counts": as_int([len(r) for r in own_rows])}


def exact(case, seed):
    s = prepare(case, seed)
    c, op = case, case["op"]
    if op == "sort":
        return _exact_sort(s["ids"], c["E"], c["align"])
    if op == "adamw":
        return _exact_adamw(s)
    plan, k, T = s["plan"], c["k"], c["T"]
    R = len(plan["sources"])
    if op in ("permute", "combine"):
        made = (plan["positions"] >= 0).reshape(-1).nonzero()[:, 0]  # choices that are made
        at, token = plan["positions"].reshape(-1).long()[made], made // k
        if op == "permute":
            if c["dtype"] == "e4m3":
                q, sc = (torch.zeros(R, t.shape[1], dtype=torch.float64, device=t.device) for t in (s["x"], s["s"]))
                q[at], sc[at] = s["x"].double()[token], s["s"].double()[token]
                return {"q": q, "s": sc}
            xs = torch.zeros(R, c["H"], dtype=torch.float64, device=at.device)
            xs[at] = s["x"].double()[token]
            dx = torch.zeros(T, c["H"], dtype=torch.float64, device=at.device).index_add_(0, token, s["dxs"].double()[at])
            return {"xs": xs, "dx": dx}
        w = s["w"].double().reshape(-1)
        y = torch.zeros(T, c["H"], dtype=torch.float64, device=at.device)
        y.index_add_(0, token, w[made, None] * s["ys"].double()[at])
        if not c["train"]:
            return {"y": y}
        dys = torch.zeros(R, c["H"], dtype=torch.float64, device=at.device)
        dys[at] = w[made, None] * s["dy"].double()[token]
        dw = torch.zeros(T * k, dtype=torch.float64, device=at.device)
        dw[made] = (s["ys"].double()[at] * s["dy"].double()[token]).sum(1)
        return {"y": y, "dys": dys, "dw": dw.reshape(T, k)}
    off = plan["offsets"].tolist()
    N, K, E = c["N"], c["K"], c["E"]
    y = torch.zeros(R, N, dtype=torch.float64, device="cuda")
    if op == "product":
        a = s["a"].double() * _spread(s["sa"].double(), K)
        for e in range(E):
            w = s["b"][e].double() * s["sb"][e].double().repeat_interleave(GROUP, 0).repeat_interleave(GROUP, 1)
            y[off[e] : off[e + 1]] = a[off[e] : off[e + 1]] @ w.t()
        return y
    dx = torch.zeros(R, K, dtype=torch.float64, device="cuda")
    dw = torch.zeros(E, N, K, dtype=torch.float64, device="cuda")
    for e in range(E):
        rows = slice(off[e], off[e + 1])
        x, dy = s["x"][rows], s["dy"][rows]
        if not len(x):
            continue
        w = _exact_quant(s["w"][e].to(torch.bfloat16), GROUP, GROUP)
        y[rows] = _exact_quant(x, 1, GROUP) @ w.t()
        dx[rows] = _exact_quant(dy, 1, GROUP, True) @ w
        dw[e] = _exact_quant(dy, GROUP, 1, True).t() @ _exact_quant(x, GROUP, 1)
    return {"y": y, "dx": dx, "dw": dw}


def _exact_codes(x, bits, positive):
    """e4m3 values of x over its group's scale, rounded down or up by the random bits; and the scales."""
    n = x.numel()
    s = _over(torch.nn.functional.pad(x, (0, -n % GROUP)).reshape(-1, GROUP).abs().amax(1)).clamp_min(LEAST)
    y = x.abs() / _spread(s, n)
    step = torch.ldexp(torch.ones_like(y), torch.frexp(y)[1].clamp_min(-5) - 4)  # the distance of e4m3's values around y
    z = (torch.floor(y / step + bits.double() / 65536.0) * step).clamp_max(448.0)
    z = torch.where(x > 0, z.clamp_min(2.0**-9), z) if positive else torch.copysign(z, x)
    return z, s


def _exact_adamw(s):
    c, lr, b1, b2, eps, step = s["case"], s["lr"], 0.9, 0.95, 1e-8, s["step"] + 1
    out = {name: x.double() for name, x in s["buffers"].items()}  # between the tensors nothing changes
    at_scale = 0
    for i, (a, n) in enumerate(s["at"]):
        p, g = s["p"][i].double(), s["g"][i].double() * s["clip"].double()
        if c["bits"] == 8:
            m, v = (x[0].double() * _spread(x[1].double(), n) for x in (s["m"][i], s["v"][i]))
            v = v * v
        else:
            m, v = s["m"][i].double(), s["v"][i].double()
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        mean, var = m / (1 - b1**step), v / (1 - b2**step)
        out["p"][a : a + n] = p - lr * c["decay"] * p - lr * mean / (var.sqrt() + eps)
        if c["bits"] == 32:
            out["m"][a : a + n], out["v"][a : a + n] = m, v
            continue
        bits, groups = _random(n, i, step, s["seed"], p.device), _ceil(n, GROUP) // GROUP
        for name, x, part, positive in (("m", m, bits & 0xFFFF, False), ("v", v.sqrt(), bits >> 16, True)):
            out[name][a : a + n], out[name + "s"][at_scale : at_scale + groups] = _exact_codes(x, part, positive)
        at_scale += groups
    return out
