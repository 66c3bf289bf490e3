"""adamw_step and AdamW against the definition in 64 bits, and the 8-bit states bit for bit.

u = 2^-24 is half a step of fp32. Every operation of the states is rounded by
itself, and the constants once: m' has 4 roundings of values at most mag(m') = |b1
m| + |c1 g|, v' 5; the update m' / d has those of m', d's (v's halved by the root, the
root, two more) and two of its own, 14 in all counted on mag(m') / d; p' two of p and
the output's. With states in 8 bits the update has an approximate reciprocal, two u
more: 16.
"""

import pytest
import torch

import thingy_b200 as tb

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
U = 2.0**-24
MASK = 0xFFFFFFFF
COMBOS = [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16),
          (torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.float16, torch.float32)]
SIZES = [1, 7, 8, 127, 128, 129, 4095, 4096, 4097, 100003, 0, 64]
HYPER = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x9E3779B9) & MASK
    x = x ^ (x >> 15)
    x = (x * 0x6A09E667) & MASK
    return x ^ (x >> 16)


def random_bits(n, ordinal, step, seed):
    key = mix((seed & MASK) ^ mix((seed >> 32) & MASK))
    key = mix(mix(key ^ (step & MASK)) ^ ordinal)
    return mix((torch.arange(n, device="cuda") * 0x9E3779B9 + key) & MASK)


def spread(s, n):
    return s.repeat_interleave(128)[:n]


def group_scales(x):
    n = x.numel()
    x = torch.where(x.isnan(), torch.zeros_like(x), x)  # NaN counts as nothing
    amax = torch.nn.functional.pad(x, (0, -n % 128)).reshape(-1, 128).abs().amax(1)
    return (amax / torch.full_like(amax, 448.0)).clamp_min(2.0**-92)


def stored(x, bits, positive):
    """Codes and scales in fp32, operation by operation."""
    s = group_scales(x)
    y = x.abs() * spread(1.0 / s, x.numel())
    up = torch.where(y < 2.0**-6, 2.0**-6, 0.0)
    z = ((y + up).view(torch.int32) + (bits << 4).int()) & -0x100000
    z = (z.view(torch.float32) - up).clamp_max(448.0)
    z = torch.where(x > 0, z.clamp_min(2.0**-9), z) if positive else z
    z = torch.where(y.isnan(), y, z)  # NaN stays, also of an infinite value over an infinite scale
    return torch.copysign(z, x if not positive else torch.ones_like(z)).to(F8), s


def tensors(sizes, p_dtype, g_dtype, seed, shift=0, gap=5):
    """Views into one buffer each, `shift` elements off its start, with gaps that must stay as they are."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    total = shift + sum(sizes) + gap * len(sizes)
    out, at = [], shift
    p = (0.5 * torch.randn(total, generator=g, device="cuda")).to(p_dtype)
    gr = (1e-2 * torch.randn(total, generator=g, device="cuda")).to(g_dtype)
    m = 1e-2 * torch.randn(total, generator=g, device="cuda")
    v = (1e-2 * torch.randn(total, generator=g, device="cuda")) ** 2
    for n in sizes:
        out.append([t[at : at + n] for t in (p, gr, m, v)])
        at += n + gap
    return (p, m, v), out


def exact(p, g, m, v, step, clip, lr, betas, eps, weight_decay):
    p, g, m, v = (t.double() for t in (p, g, m, v))
    g = g * clip
    b1, b2 = betas
    size = (b1 * m).abs() + ((1 - b1) * g).abs()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    rate, d = lr / (1 - b1**step), (v / (1 - b2**step)).sqrt() + eps
    return p * (1 - lr * weight_decay) - rate * m / d, m, v, size, rate * size / d


@pytest.mark.parametrize("shift", [0, 1, 4])
@pytest.mark.parametrize("p_dtype,g_dtype", COMBOS)
def test_step_in_32_bits(p_dtype, g_dtype, shift):
    buffers, parts = tensors(SIZES, p_dtype, g_dtype, 3, shift)
    before = [b.clone() for b in buffers]
    clip = torch.full((1,), 0.625, device="cuda")
    want = [exact(*t, 7, 0.625, **HYPER) for t in parts]
    p0 = [t[0].clone() for t in parts]
    tb.adamw_step(*map(list, zip(*parts)), step=7, grad_scale=clip, **HYPER)
    for (p, _, m, v), old, (wp, wm, wv, size, update) in zip(parts, p0, want):
        assert bool(((m.double() - wm).abs() <= 4 * U * size).all())
        assert bool(((v.double() - wv).abs() <= 5 * U * wv).all())
        info = torch.finfo(p_dtype)
        tol = 14 * U * update + 3 * U * old.double().abs() + half_step(p_dtype) * wp.abs() * 1.0001 + info.tiny * info.eps
        assert bool(((p.double() - wp).abs() <= tol).all())
    kept = torch.ones_like(before[0], dtype=torch.bool)
    at = shift
    for n in SIZES:
        kept[at : at + n] = False
        at += n + 5
    for b, old in zip(buffers, before):  # gaps
        assert torch.equal(b[kept], old[kept])


@pytest.mark.parametrize("shift", [0, 1, 8])
@pytest.mark.parametrize("p_dtype,g_dtype", COMBOS)
def test_step_in_8_bits(p_dtype, g_dtype, shift):
    """Codes and scales are those of the formula; parameters within rounding of 64 bits."""
    _, parts = tensors(SIZES, p_dtype, g_dtype, 4, shift)
    seed, step, clip = 0x123456789ABCDEF, 12, torch.full((1,), 0.5, device="cuda")
    states = []
    for i, (_, _, m, v) in enumerate(parts):
        zero = torch.full_like(m, 32768, dtype=torch.int64)
        places = []
        for x, positive in ((m, False), (v.sqrt(), True)):
            codes, scales = stored(x, zero, positive)
            place = torch.zeros(x.numel() + shift, dtype=torch.uint8, device="cuda").view(F8)[shift:]
            place.copy_(codes)
            places.append((place, scales))
        states.append(places)
    p0 = [t[0].clone() for t in parts]
    old = [[(q.float() * spread(s, q.numel())) for q, s in pair] for pair in states]
    tb.adamw_step([t[0] for t in parts], [t[1] for t in parts], [s[0] for s in states], [s[1] for s in states], step=step,
                  seed=seed, grad_scale=clip, **HYPER)
    b1, b2 = HYPER["betas"]
    for i, ((p, g, _, _), (m, r), ((mq, ms), (vq, vs)), before) in enumerate(zip(parts, old, states, p0)):
        bits = random_bits(p.numel(), i, step, seed)
        gc = g.float() * 0.5
        m32, v32 = b1 * m + (1.0 - b1) * gc, b2 * (r * r) + (1.0 - b2) * (gc * gc)
        wp, _, _, _, update = exact(before, g, m, r.double() ** 2, step, 0.5, **HYPER)
        for (q, sc), (wq, ws) in (((mq, ms), stored(m32, bits & 0xFFFF, False)), ((vq, vs), stored(torch.sqrt(v32), bits >> 16, True))):
            assert torch.equal(q.view(torch.uint8), wq.view(torch.uint8))
            assert torch.equal(sc, ws)
        info = torch.finfo(p_dtype)
        tol = 16 * U * update + 3 * U * before.double().abs() + half_step(p_dtype) * wp.abs() * 1.0001 + info.tiny * info.eps
        assert bool(((p.double() - wp).abs() <= tol).all())


@pytest.mark.parametrize("scale", [1e-19, 1e-16, 3e-15, 1.0, 3e14, 1e18])
def test_codes_at_the_ends_of_the_range(scale):
    """Roots from subnormal second moments to large ones, zeros among them: both forms of the square root."""
    n = 1 << 18
    gen = torch.Generator(device="cuda").manual_seed(11)
    g = scale * torch.randn(n, generator=gen, device="cuda") * torch.exp(2.0 * torch.randn(n, generator=gen, device="cuda"))
    g[torch.rand(n, generator=gen, device="cuda") < 0.01] = 0.0
    g[256:384] = 0.0
    p, m, v = torch.zeros(n, device="cuda"), tb.adamw_state(g, 8), tb.adamw_state(g, 8)
    old_m, old_r = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    for step in (1, 2, 3):
        tb.adamw_step([p], [g], [m], [v], step=step, lr=0.0, betas=(0.9, 0.95), seed=17)
        bits = random_bits(n, 0, step, 17)
        m32, v32 = 0.9 * old_m + (1.0 - 0.9) * g, 0.95 * (old_r * old_r) + (1.0 - 0.95) * (g * g)
        for (q, sc), (wq, ws) in ((m, stored(m32, bits & 0xFFFF, False)), (v, stored(torch.sqrt(v32), bits >> 16, True))):
            assert torch.equal(q.view(torch.uint8), wq.view(torch.uint8)) and torch.equal(sc, ws)
        old_m, old_r = (q.float() * spread(sc, n) for q, sc in (m, v))


def test_codes_are_neighbours_and_their_mean_is_kept():
    """Each code is one of the two around the value in 64 bits; over many elements the error's mean vanishes."""
    n = 1 << 20
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(n, generator=g, device="cuda")
    p, zeros = torch.zeros(n, device="cuda"), tb.adamw_state(x, 8)
    m, v = tb.adamw_state(x, 8), zeros
    tb.adamw_step([p], [x], [m], [v], step=1, lr=0.0, betas=(0.5, 0.5), seed=5)
    for (q, s), want in ((m, 0.5 * x.double()), (v, (0.5 * x.double() ** 2).sqrt())):
        y = want.abs() / spread(s.double(), n)
        step = torch.ldexp(torch.ones_like(y), torch.frexp(y)[1].clamp_min(-5) - 4)
        off = (q.double().abs() - y) / step
        assert bool((off.abs() <= 1 + 2.0**-18).all())  # fp32 values of 2^4 steps of 2^20 a code
        # uniform bits: a variance of f (1 - f) <= 1/4 a code; the mean within six of its deviations and 2^-16
        assert abs(float(off.mean())) <= 6 * 0.5 / n**0.5 + 2.0**-16


def test_small_moments_decay():
    """A second moment far above its gradients decays as b2^t although its codes are 2^-3 apart."""
    n, steps, b2 = 1 << 16, 200, 0.99
    p, m = torch.zeros(n, device="cuda"), tb.adamw_state(torch.zeros(n, device="cuda"), 8)
    v = tb.adamw_state(torch.zeros(n, device="cuda"), 8)
    big = torch.ones(n, device="cuda")
    tb.adamw_step([p], [big], [m], [v], step=1, lr=0.0, betas=(0.9, b2), seed=1)
    none = torch.zeros(n, device="cuda")
    for t in range(2, steps + 2):
        tb.adamw_step([p], [none], [m], [v], step=t, lr=0.0, betas=(0.9, b2), seed=1)
    got = float((v[0].double() * spread(v[1].double(), n)).mean())
    # r decays by sqrt(b2) a step in the mean; each step's rounding moves the mean of n codes by at most
    # 2^-4 r / sqrt(n) (one deviation), and cutting the random bits to 16 by 2^-17 of a code downwards
    want = (1 - b2) ** 0.5 * b2 ** (steps / 2)
    assert abs(got / want - 1) <= 6 * 2.0**-4 / n**0.5 * steps**0.5 + steps * 2.0**-19


def test_codes_of_zeros_and_of_extremes():
    n = 384
    g = torch.zeros(n, device="cuda")
    g[128:256] = 1e-25  # below the least scale's codes for r, far below for m
    g[130] = 1e-30
    g[256] = float("inf")
    g[300] = 1.0
    p, m, v = torch.zeros(n, device="cuda"), tb.adamw_state(g, 8), tb.adamw_state(g, 8)
    tb.adamw_step([p], [g], [m], [v], step=1, lr=1.0, seed=2)
    assert bool((m[0][:128].float() == 0).all()) and bool((v[0][:128].float() == 0).all()) and bool((p[:128] == 0).all())
    assert float(m[1][0]) == float(v[1][0]) == 2.0**-92
    assert bool((v[0][128:256].float() >= 0).all())
    assert bool(torch.isfinite(p[:256]).all())
    assert bool(torch.isnan(m[0][256].float()))
    q = torch.full((n,), float("nan"), device="cuda")
    q[5] = 2.0
    m, v = tb.adamw_state(q, 8), tb.adamw_state(q, 8)
    tb.adamw_step([torch.zeros(n, device="cuda")], [q], [m], [v], step=1, lr=1.0)
    keep = torch.isnan(m[0].float())
    assert int(keep.sum()) == n - 1 and not bool(keep[5])


def test_a_lost_code_divides_by_no_eps():
    """An element whose root is far below its group's keeps the least code, not zero."""
    n = 128
    g = torch.full((n,), 1e-6, device="cuda")
    g[0] = 1.0
    p, m, v = torch.zeros(n, device="cuda"), tb.adamw_state(g, 8), tb.adamw_state(g, 8)
    tb.adamw_step([p], [g], [m], [v], step=1, lr=0.0, seed=3)
    assert bool((v[0].float() > 0).all())


@pytest.mark.parametrize("count", [1, 40, 41, 480, 481, 1000])
@pytest.mark.parametrize("bits", [8, 32])
def test_lists_of_any_length(count, bits):
    sizes = [(37 * i) % 300 for i in range(count)]
    g = torch.Generator(device="cuda").manual_seed(count)
    p = [torch.randn(n, generator=g, device="cuda") for n in sizes]
    gr = [torch.randn(n, generator=g, device="cuda") for n in sizes]
    one = [t.clone() for t in p]
    m, v = ([tb.adamw_state(t, bits) for t in p] for _ in range(2))
    tb.adamw_step(p, gr, m, v, step=1, lr=0.1, seed=9)
    for i, n in enumerate(sizes):
        if n:
            want = exact(one[i], gr[i], torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), 1, 1.0, 0.1, (0.9, 0.999), 1e-8, 0.0)
            assert bool(((p[i].double() - want[0]).abs() <= 16 * U * want[4] + 4 * U * (one[i].double().abs() + want[0].abs())).all())
        if bits == 8:
            m32 = 0.1 * gr[i]
            # c1 = 1 - 0.9 in 64 bits, rounded
            wq, ws = stored((1.0 - 0.9) * gr[i], random_bits(n, i, 1, 9) & 0xFFFF, False)
            assert torch.equal(m[i][0].view(torch.uint8), wq.view(torch.uint8)) and torch.equal(m[i][1], ws)


def test_large_tensor():
    """More elements than a launch's first wave, and offsets past 2^31 bytes."""
    n = (1 << 29) + 12345
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g[-1], g[n // 2], g[0] = 1.0, -1.0, 2.0
    m, v = tb.adamw_state(p, 32), tb.adamw_state(p, 32)
    tb.adamw_step([p], [g], [m], [v], step=1, lr=0.5)
    assert int((p != 0).sum()) == 3
    assert float(p[-1]) == -0.5 and float(p[n // 2]) == 0.5 and float(p[0]) == -0.5
    assert float(v[-1]) == float(torch.tensor(1.0 - 0.999))


def test_step_and_rate_on_the_gpu():
    """Captured and replayed with a step and a rate that change; near the host's values."""
    n, steps = 3000, 4
    gen = torch.Generator(device="cuda").manual_seed(6)
    p0 = torch.randn(n, generator=gen, device="cuda")
    grads = [torch.randn(n, generator=gen, device="cuda") for _ in range(steps)]
    rates = [0.1, 0.05, 0.2, 0.025]
    host = [p0.clone(), tb.adamw_state(p0, 8), tb.adamw_state(p0, 8)]
    gpu = [p0.clone(), tb.adamw_state(p0, 8), tb.adamw_state(p0, 8)]
    count, rate = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(1, device="cuda")
    place = torch.zeros(n, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        count.add_(1)
        tb.adamw_step([gpu[0]], [place], [gpu[1]], [gpu[2]], step=count, lr=rate, seed=4)
    for t in range(steps):
        tb.adamw_step([host[0]], [grads[t]], [host[1]], [host[2]], step=t + 1, lr=rates[t], seed=4)
        place.copy_(grads[t])
        rate.fill_(rates[t])
        graph.replay()
        for a, b in zip(host[1] + host[2], gpu[1] + gpu[2]):
            assert torch.equal(a, b)  # moments do not depend on the corrections
        # three factors rounded in other ways, each at most one step of 2^-23, on updates of at most 4 rates
        assert bool(((host[0] - gpu[0]).abs() <= (t + 1) * (12 * U * 4 * 0.2 + 2 * U * host[0].abs().max())).all())


def test_repeats():
    _, parts = tensors([5000, 77], torch.bfloat16, torch.float32, 8)
    runs = []
    for seed in (1, 1, 2):
        p, m, v = ([t[0].clone() for t in parts], [tb.adamw_state(t[0], 8) for t in parts], [tb.adamw_state(t[0], 8) for t in parts])
        tb.adamw_step(p, [t[1] for t in parts], m, v, step=3, lr=0.1, seed=seed)
        runs.append([x.view(torch.uint8) if x.dtype == F8 else x for pair in m + v for x in pair] + p)
    assert all(torch.equal(a, b) for a, b in zip(runs[0], runs[1]))
    assert not all(torch.equal(a, b) for a, b in zip(runs[0], runs[2]))


def test_gradients_of_other_strides():
    g = torch.randn(60, 40, device="cuda")
    p = [torch.randn(40, 60, device="cuda")]
    q = [p[0].clone()]
    states = [[torch.zeros(40, 60, device="cuda")] for _ in range(4)]
    tb.adamw_step(p, [g.t()], states[0], states[1], step=1, lr=0.1)
    tb.adamw_step(q, [g.t().contiguous()], states[2], states[3], step=1, lr=0.1)
    assert torch.equal(p[0], q[0])
    e = torch.ones(1, device="cuda").expand(40, 60)
    tb.adamw_step(p, [e], states[0], states[1], step=2, lr=0.1)


def test_optimizer_against_torch_in_64_bits():
    torch.manual_seed(0)
    shapes, steps = [(64, 128), (5,), ()], 6
    start = [torch.randn(s) for s in shapes]
    mine = [t.clone().cuda().requires_grad_() for t in start]
    theirs = [t.clone().double().requires_grad_() for t in start]
    args = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    a, b = tb.AdamW(mine, **args), torch.optim.AdamW(theirs, **args)
    for t in range(steps):
        for x, y in zip(mine, theirs):
            g = torch.randn(x.shape)
            x.grad, y.grad = g.cuda(), g.double()
        if t == 3:
            mine[1].grad = theirs[1].grad = None  # a parameter of another age from here on
        a.step(), b.step()
    for x, y in zip(mine, theirs):
        # updates of at most 4 rates (mag(m') / d <= 0.1 sum 0.9^i / sqrt(0.01) and less), errors carried in m and v
        tol = steps * (steps * 20 * U * 4 * args["lr"] + 4 * U * (y.abs() + 1))
        assert bool(((x.detach().double().cpu() - y.detach()).abs() <= tol.detach()).all())


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("capturable", [False, True])
def test_optimizer_states_are_stored_and_loaded(bits, capturable):
    torch.manual_seed(1)
    start = [torch.randn(300, device="cuda").bfloat16(), torch.randn(129, device="cuda")]
    grads = [[torch.randn_like(p) for p in start] for _ in range(5)]

    def run(opt, params, which):
        for t in which:
            for p, g in zip(params, grads[t]):
                p.grad = g if not (t == 1 and p.numel() == 129) else None
            opt.step()

    whole = [p.clone().requires_grad_() for p in start]
    opt = tb.AdamW(whole, state_bits=bits, capturable=capturable, seed=3)
    run(opt, whole, range(5))
    first = [p.clone().requires_grad_() for p in start]
    opt1 = tb.AdamW(first, state_bits=bits, capturable=capturable, seed=3)
    run(opt1, first, range(3))
    saved = opt1.state_dict()
    second = [p.detach().clone().requires_grad_() for p in first]
    opt2 = tb.AdamW(second, state_bits=bits, capturable=capturable)
    opt2.load_state_dict(saved)
    for p, q in zip(first, second):
        for name, value in opt1.state[p].items():
            other = opt2.state[q][name]
            if isinstance(value, torch.Tensor):
                assert other.dtype == value.dtype and other.data_ptr() != value.data_ptr()
    run(opt2, second, range(3, 5))
    for p, q in zip(whole, second):
        assert torch.equal(p, q)
    assert [int(opt.state[p]["step"]) for p in whole] == [5, 4]


def test_optimizer_captured():
    torch.manual_seed(2)
    p = torch.randn(500, device="cuda")
    eager, captured = p.clone().requires_grad_(), p.clone().requires_grad_()
    grads = [torch.randn(500, device="cuda") for _ in range(4)]
    a = tb.AdamW([eager], lr=0.1, state_bits=8, capturable=True)
    b = tb.AdamW([captured], lr=0.1, state_bits=8, capturable=True)
    captured.grad = grads[0].clone()
    with pytest.raises(RuntimeError, match="one step before"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            b.step()
    b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.step()
    for t in range(4):
        eager.grad = grads[t]
        a.step()
        if t:
            captured.grad.copy_(grads[t])
            graph.replay()
        assert torch.equal(eager, captured)


def test_optimizer_captured_without_a_gradient():
    """Parameters that would part company within a graph: refused, and nothing has changed."""
    ps = [torch.randn(10, device="cuda", requires_grad=True) for _ in range(2)]
    opt = tb.AdamW(ps, lr=0.1, capturable=True)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    ps[1].grad = None
    before = [p.detach().clone() for p in ps]
    with pytest.raises(RuntimeError, match="same steps"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, before))
    assert [int(opt.state[p]["step"]) for p in ps] == [1, 1]
    opt.step()  # eager: they part
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    assert [int(opt.state[p]["step"]) for p in ps] == [3, 1]


def test_version_counters_see_the_step():
    p = torch.randn(8, device="cuda", requires_grad=True)
    y = (p * p).sum()
    tb.adamw_step([p], [torch.ones(8, device="cuda")], [tb.adamw_state(p)], [tb.adamw_state(p)], step=1, lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals():
    p, g = torch.zeros(200, device="cuda"), torch.zeros(200, device="cuda")
    m, v = tb.adamw_state(p), tb.adamw_state(p)
    m8, v8 = tb.adamw_state(p, 8), tb.adamw_state(p, 8)
    step = tb.adamw_step
    for call, match in [
        (lambda: step([p], [g], [m], [v], step=0, lr=0.1), "counts from 1"),
        (lambda: step([p], [g], [m], [v], step=1, lr=-0.1), "lr"),
        (lambda: step([p], [g], [m], [v], step=1, lr=float("nan")), "lr"),
        (lambda: step([p], [g], [m], [v], step=1, lr=0.1, betas=(1.0, 0.9)), "betas"),
        (lambda: step([p], [g], [m], [v], step=1, lr=0.1, betas=(0.9, float("nan"))), "betas"),
        (lambda: step([p], [g], [m], [v], step=1, lr=0.1, eps=-1.0), "eps"),
        (lambda: step([p], [g], [m], [v], step=1, lr=0.1, weight_decay=-1.0), "weight_decay"),
        (lambda: step([p, p], [g, g], [m, tb.adamw_state(p)], [v, tb.adamw_state(p)], step=1, lr=0.1), "params must not overlap"),
        (lambda: step([p, torch.zeros_like(p)], [g, g], [m, m], [v, tb.adamw_state(p)], step=1, lr=0.1), "exp_avgs must not overlap"),
        (lambda: step([p], [g], [m], [m], step=1, lr=0.1), "share memory"),
        (lambda: step([p], [g], [p], [v], step=1, lr=0.1), "share memory"),
        (lambda: step([p], [g], [m8], [(v8[0], m8[1])], step=1, lr=0.1), "share memory"),
        (lambda: step([p, torch.zeros_like(p)], [g, g], [m8, (tb.adamw_state(p, 8)[0], m8[1])], [v8, tb.adamw_state(p, 8)], step=1,
                      lr=0.1), "scales must not overlap"),
        (lambda: step([p], [g], [m], [v, v], step=1, lr=0.1), "same length"),
        (lambda: step([p], [g[:100]], [m], [v], step=1, lr=0.1), "shapes"),
        (lambda: step([p], [None], [m], [v], step=1, lr=0.1), "hold tensors"),
        (lambda: step(3, [g], [m], [v], step=1, lr=0.1), "sequence"),
        (lambda: step([p[::2]], [g[::2]], [m[:100]], [v[:100]], step=1, lr=0.1), "contiguous"),
        (lambda: step([p.cpu()], [g], [m], [v], step=1, lr=0.1), "CUDA"),
        (lambda: step([p.double()], [g], [m], [v], step=1, lr=0.1), "bfloat16, float16 or float32"),
        (lambda: step([p], [g.half()], [m], [v], step=1, lr=0.1), "dtype"),
        (lambda: step([p, p.half()], [g, g], [m, m], [v, v], step=1, lr=0.1), "one dtype"),
        (lambda: step([p], [g], [m.bfloat16()], [v], step=1, lr=0.1), "float32"),
        (lambda: step([p], [g], [m8], [v], step=1, lr=0.1), "all pairs"),
        (lambda: step([p], [g], [(m8[0], m8[1][:1])], [v8], step=1, lr=0.1), "scales"),
        (lambda: step([p], [g], [(m8[0][:100], m8[1])], [v8], step=1, lr=0.1), "codes"),
        (lambda: step([p], [g], [m], [v], step=torch.ones(1, device="cuda"), lr=0.1), "int64"),
        (lambda: step([p], [g], [m], [v], step=1, lr=torch.ones(2, device="cuda")), "float32"),
        (lambda: step([p], [g], [m], [v], step=1, lr=0.1, grad_scale=torch.ones(1)), "grad_scale"),
        (lambda: tb.adamw_state(p, 4), "32 or 8"),
        (lambda: tb.AdamW([p], state_bits=16), "state_bits"),
        (lambda: tb.AdamW([p], lr=-1.0), "lr"),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
    assert bool((p == 0).all())
    step([], [], [], [], step=1, lr=0.1)
