"""The mixture-of-experts layer for few tokens, against its definition in 64 bits.

The router's logits are sums of exact products: |err| <= H 2^-23 of the sum of
magnitudes, so a choice is checked exactly only for the tokens whose logits
(or biased scores) are separated by more than that. Hidden rows are cast to e4m3: an
fp32 error of the sums moves a code near a rounding boundary by one step, 2^-3
of the element at most, for a share of the elements of about (128 + KB) 2^-23
/ 2^-4; the outputs carry that as a random sum. Tolerance on the output:
2^-8 |ref| (bf16) + 2^-3 / sqrt(I) of the row's magnitude for at most one moved
code in sqrt(I) of them (far above what the shares give), i.e. rms(row) / 8.
The relative 2-norm of a row is held to 2^-8.
"""

import pytest
import torch

import thingy_b200 as tb
from thingy_b200.moe import quantize_experts

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def _inputs(T, E, H, I, seed, layout="row"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, H, generator=g, device="cuda")
    x[:, ::97] *= 20.0
    x = x.to(torch.bfloat16)
    w = (1.0 + 0.1 * torch.randn(H, generator=g, device="cuda")).to(torch.bfloat16)
    q, s, _, n = tb.rms_norm_fp8(x, w, 1e-6, scale_layout=layout, return_normalized=True)
    router = (0.05 * torch.randn(E, H, generator=g, device="cuda")).to(torch.bfloat16)
    w13 = quantize_experts((0.03 * torch.randn(E, 2 * I, H, generator=g, device="cuda")).to(torch.bfloat16))
    w2 = quantize_experts((0.03 * torch.randn(E, H, I, generator=g, device="cuda")).to(torch.bfloat16))
    return n, q, s, router, *w13, *w2


def _spread(s, R, C):
    return s.double().repeat_interleave(128, -2)[..., :R, :].repeat_interleave(128, -1)[..., :C]


def _reference(x, q, s, router, w13, s13, w2, s2, k, scoring, renormalize=True, routed_scale=1.0, bias=None):
    T, H = x.shape
    E, _, I = w2.shape
    logits = x.double() @ router.double().t()
    p = torch.softmax(logits, 1) if scoring == "softmax" else torch.sigmoid(logits)
    sel = logits if bias is None else p + bias.double()
    top, ids = torch.sort(sel, dim=1, descending=True, stable=True)
    # tokens whose choice no fp32 rounding can change: order inside the k and the step after them
    sure = (top[:, :-1] - top[:, 1:])[:, :k].amin(1) > 1e-5 if E > 1 else torch.ones(T, dtype=torch.bool, device=x.device)
    ids = ids[:, :k]
    w = p.gather(1, ids)
    if renormalize:
        w = w / w.sum(1, keepdim=True)
    w = w * routed_scale
    a = q.double() * s.double().repeat_interleave(128, 1)
    y = torch.zeros(T, H, dtype=torch.float64, device=x.device)
    for e in range(E):
        t, j = (ids == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        gu = a[t] @ (w13[e].double() * _spread(s13[e], 2 * I, H)).t()
        h = torch.nn.functional.silu(gu[:, :I]) * gu[:, I:]
        sh = (h.abs().view(len(t), -1, 128).amax(2) / 448.0).clamp_min(1e-4).float().double().repeat_interleave(128, 1)
        h = (h / sh).float().to(F8).double() * sh
        y[t] += w[t, j, None] * (h @ (w2[e].double() * _spread(s2[e], H, I)).t())
    return y, ids, w, sure


def _check(got, ref):
    got = got.double()
    rms = ref.pow(2).mean(1, keepdim=True).sqrt()
    assert bool(((got - ref).abs() <= ref.abs() * 2.0**-8 + rms / 8 + 1e-30).all())
    rel = (got - ref).norm(dim=1) / ref.norm(dim=1)
    assert rel.max().item() <= 2.0**-8, rel.max().item()


CASES = [  # T, E, k, H, I
    (1, 1, 1, 128, 128),
    (1, 8, 2, 256, 128),
    (1, 128, 8, 1024, 384),
    (2, 4, 4, 384, 256),
    (7, 8, 2, 1152, 640),
    (8, 60, 4, 2048, 128),
    (9, 64, 6, 640, 256),
    (16, 3, 1, 512, 512),
    (17, 16, 3, 896, 256),
    (31, 256, 8, 768, 128),
    (32, 5, 2, 7168, 256),
    (33, 40, 5, 1280, 384),
    (64, 512, 16, 256, 128),
    (64, 1, 1, 512, 256),
    (64, 2, 2, 2944, 128),
    (64, 64, 6, 2048, 512),
]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,H,I", CASES)
def test_layer(T, E, k, H, I, scoring):
    ops = _inputs(T, E, H, I, seed=T + E + k + H, layout="col" if T % 2 else "row")
    ids = torch.full((T, k), -1, dtype=torch.int32, device="cuda")
    weights = torch.full((T, k), -1.0, device="cuda")
    y = tb.moe_fp8(*ops, top_k=k, scoring=scoring, topk_ids=ids, topk_weights=weights)
    ref, rid, rw, sure = _reference(*ops, k, scoring)
    assert sure.float().mean() > 0.8
    assert torch.equal(ids.long()[sure], rid[sure])
    assert torch.allclose(weights.double()[sure], rw[sure], rtol=1e-4, atol=0)
    _check(y[sure], ref[sure])
    assert tb_device_error() == 0


def tb_device_error():
    from thingy_b200 import _lib

    return _lib.device_error()


@pytest.mark.parametrize("T", [3, 20])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_bias_scale_and_plain_scores(T, scoring, renormalize):
    ops = _inputs(T, 32, 512, 256, seed=T)
    bias = 0.3 * torch.randn(32, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    kw = dict(scoring=scoring, renormalize=renormalize, routed_scale=2.5, bias=bias)
    ids = torch.empty(T, 5, dtype=torch.int32, device="cuda")
    y = tb.moe_fp8(*ops, top_k=5, topk_ids=ids, **kw)
    ref, rid, _, sure = _reference(*ops, 5, **kw)
    assert sure.float().mean() > 0.8
    assert torch.equal(ids.long()[sure], rid[sure])
    _check(y[sure], ref[sure])


@pytest.mark.parametrize("T", [2, 30])
def test_ties_go_to_the_lowest_expert(T):
    ops = list(_inputs(T, 40, 256, 128, seed=3))
    ops[3] = ops[3][:1].expand(40, 256).contiguous()  # every logit the same
    ids = torch.empty(T, 6, dtype=torch.int32, device="cuda")
    weights = torch.empty(T, 6, device="cuda")
    tb.moe_fp8(*ops, top_k=6, topk_ids=ids, topk_weights=weights)
    assert torch.equal(ids.cpu(), torch.arange(6, dtype=torch.int32).expand(T, 6))
    assert torch.allclose(weights, torch.full_like(weights, 1 / 6))


@pytest.mark.parametrize("T", [4, 20])
def test_nonfinite_logits_keep_to_their_token(T):
    ops = list(_inputs(T, 16, 256, 128, seed=5))
    want = tb.moe_fp8(*ops, top_k=3)
    x = ops[0].clone()
    x[1, 7] = float("nan")
    x[2, 9] = float("inf")
    ids = torch.empty(T, 3, dtype=torch.int32, device="cuda")
    y = tb.moe_fp8(x, *ops[1:], top_k=3, topk_ids=ids)
    rest = [t for t in range(T) if t not in (1, 2)]
    # the active experts differ, and with them where items are split over K
    _check(y[rest], want[rest].double())
    assert torch.isnan(y[1]).all()
    assert bool(((ids >= 0) & (ids < 16)).all())
    for row in ids.tolist():
        assert len(set(row)) == 3


def test_zero_rows_and_large_values():
    ops = list(_inputs(5, 8, 256, 256, seed=6))
    q = ops[1].clone()
    q[2] = 0.0  # a token of zeros: its hidden rows and outputs are zero
    ops[1] = q
    y = tb.moe_fp8(*ops, top_k=2)
    assert bool((y[2] == 0).all())
    s = ops[2].clone()
    s[3] *= 1e4  # gates far outside exp's range
    ops[2] = s
    y = tb.moe_fp8(*ops, top_k=2)
    ref, *_ = _reference(*ops, 2, "softmax")
    _check(y[[0, 1, 3, 4]], ref[[0, 1, 3, 4]])


def test_repeats_streams_graphs_and_shared_workspace():
    a = _inputs(6, 24, 1024, 256, seed=7)
    b = _inputs(40, 10, 512, 384, seed=8)
    wa, wb = tb.moe_fp8(*a, top_k=4), tb.moe_fp8(*b, top_k=2, scoring="sigmoid")
    ws = tb.moe_workspace(64, 24, 4, 1024, 384)
    for _ in range(5):
        assert torch.equal(tb.moe_fp8(*a, top_k=4, workspace=ws), wa)
        assert torch.equal(tb.moe_fp8(*b, top_k=2, scoring="sigmoid", workspace=ws), wb)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ya = tb.moe_fp8(*a, top_k=4)
    yb = tb.moe_fp8(*b, top_k=2, scoring="sigmoid")
    torch.cuda.synchronize()
    assert torch.equal(ya, wa) and torch.equal(yb, wb)
    out = torch.empty_like(wa)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tb.moe_fp8(*a, top_k=4, out=out)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, wa)


def test_strided_rows_and_out():
    ops = list(_inputs(12, 8, 512, 128, seed=9))
    want = tb.moe_fp8(*ops, top_k=2)
    x = torch.zeros(12, 1024, dtype=torch.bfloat16, device="cuda")
    x[:, 256:768] = ops[0]
    q = torch.zeros(12, 1024, dtype=F8, device="cuda")
    q[:, 256:768] = ops[1]
    out = torch.full((12, 528), 3.0, dtype=torch.bfloat16, device="cuda")
    tb.moe_fp8(x[:, 256:768], q[:, 256:768], *ops[2:], top_k=2, out=out[:, 8:520])
    assert torch.equal(out[:, 8:520], want)
    assert bool((out[:, :8] == 3).all()) and bool((out[:, 520:] == 3).all())


def test_no_tokens():
    ops = _inputs(2, 8, 256, 128, seed=1)
    y = tb.moe_fp8(*(t[:0] for t in ops[:3]), *ops[3:], top_k=2)
    assert y.shape == (0, 256)


def test_refusals():
    ops = list(_inputs(4, 8, 256, 128, seed=1))

    def call(i=None, t=None, **kw):
        args = list(ops)
        if i is not None:
            args[i] = t
        return tb.moe_fp8(*args, **{"top_k": 2, **kw})

    with pytest.raises(ValueError, match="top_k"):
        call(top_k=9)
    with pytest.raises(ValueError, match="top_k"):
        call(top_k=0)
    with pytest.raises(ValueError, match="scoring"):
        call(scoring="tanh")
    with pytest.raises(ValueError, match="at most 64"):
        big = _inputs(65, 8, 256, 128, seed=1)
        tb.moe_fp8(*big, top_k=2)
    with pytest.raises(ValueError, match="bfloat16"):
        call(0, ops[0].float())
    with pytest.raises(ValueError, match="router"):
        call(3, ops[3].float())
    with pytest.raises(ValueError, match="w13"):
        call(4, ops[4][:, :128])
    with pytest.raises(ValueError, match="w2_scale"):
        call(7, ops[7][:4])
    with pytest.raises(ValueError, match="contiguous"):
        call(6, ops[6].transpose(1, 2).contiguous().transpose(1, 2))
    with pytest.raises(ValueError, match="float32"):
        call(2, ops[2].half())
    with pytest.raises(ValueError, match="workspace"):
        call(workspace=torch.zeros(256, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="bias"):
        call(bias=torch.zeros(7, device="cuda"))
    with pytest.raises(ValueError, match="topk_ids"):
        call(topk_ids=torch.zeros(4, 2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="multiples of 128"):
        quantize_experts(torch.zeros(2, 100, 128, dtype=torch.bfloat16, device="cuda"))
