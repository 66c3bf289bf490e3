"""Tensors of an AdamW step that share memory in any way are refused, and nothing has changed."""

import pytest
import torch

import thingy_b200 as tb

pytestmark = pytest.mark.gpu
N = 256


def fresh(bits):
    g = torch.Generator(device="cuda").manual_seed(1)
    p = [torch.randn(N, generator=g, device="cuda") for _ in range(2)]
    grads = [torch.randn(N, generator=g, device="cuda") for _ in range(2)]
    return p, grads, [tb.adamw_state(t, bits) for t in p], [tb.adamw_state(t, bits) for t in p]


def overlapping(elements, dtype=torch.float32):
    """Two tensors of N elements that share `elements`."""
    flat = torch.zeros((2 * N - elements) * dtype.itemsize, dtype=torch.uint8, device="cuda").view(dtype)
    return flat[:N], flat[N - elements :]


def parts(*lists):
    return [t for one in lists for x in one for t in (x if isinstance(x, tuple) else (x,))]


CASES = ["p p", "m m", "v v", "p0 m0", "p0 v0", "m0 v0", "p0 m1", "p1 m0", "m0 v1", "m1 v0", "p1 v0", "p0 g0", "p0 g1", "g0 m1", "v1 g0"]


@pytest.mark.parametrize("shared", [1, 100, N])
@pytest.mark.parametrize("case", CASES)
def test_states_in_32_bits(case, shared):
    lists = dict(zip("pgmv", fresh(32)))
    a, b = overlapping(shared)
    for place, t in zip((case if "0" in case or "1" in case else f"{case[0]}0 {case[0]}1").split(), (a, b)):
        lists[place[0]][int(place[1])] = t
    before = [t.clone() for t in parts(*lists.values())]
    with pytest.raises(ValueError, match="overlap|share memory"):
        tb.adamw_step(*lists.values(), step=1, lr=0.1)
    assert all(torch.equal(t, o) for t, o in zip(parts(*lists.values()), before))


@pytest.mark.parametrize("kind", ["codes", "scales", "codes and scales", "param and codes", "param and scales", "grad and codes"])
@pytest.mark.parametrize("other", [0, 1])
def test_states_in_8_bits(kind, other):
    p, g, m, v = fresh(8)
    flat = torch.zeros(4 * N, dtype=torch.uint8, device="cuda")
    code, scale = flat[: N].view(torch.float8_e4m3fn), flat[:8].view(torch.float32)
    if kind == "codes":
        m[0] = (code, m[0][1])
        v[other] = (flat[N - 1 : 2 * N - 1].view(torch.float8_e4m3fn), v[other][1])
    elif kind == "scales":
        m[0], v[other] = (m[0][0], flat[:8].view(torch.float32)), (v[other][0], flat[4:12].view(torch.float32))
    elif kind == "codes and scales":
        m[0] = (code, m[0][1])
        v[other] = (v[other][0], flat[N - 4 : N + 4].view(torch.float32))
    elif kind == "param and codes":
        p[0], m[other] = flat.view(torch.float32), (code, m[other][1])
    elif kind == "param and scales":
        p[0], m[other] = flat.view(torch.float32), (m[other][0], scale)
    else:
        g[0], v[other] = flat.view(torch.float32), (code, v[other][1])
    before = [t.clone() for t in parts(p, g, m, v)]
    with pytest.raises(ValueError, match="overlap|share memory"):
        tb.adamw_step(p, g, m, v, step=1, lr=0.1)
    assert all(torch.equal(t.view(torch.uint8), o.view(torch.uint8)) for t, o in zip(parts(p, g, m, v), before))


def test_neighbours_in_any_order_are_taken():
    """Parts of one buffer that touch, in orders that have to be sorted and merged; a gradient for two parameters."""
    g = torch.Generator(device="cuda").manual_seed(2)
    sizes = [5, 256, 1, 64, 33, 128, 7, 300]
    flat = torch.rand(3 * sum(sizes), generator=g, device="cuda")
    lists = ([], [], [])
    pieces = [(n, k) for n in sizes for k in range(3)]
    order = torch.randperm(len(pieces), generator=torch.Generator().manual_seed(3)).tolist()
    starts, at = {}, 0
    for i in order:
        starts[i] = at
        at += pieces[i][0]
    for i, (n, k) in enumerate(pieces):
        lists[k].append(flat[starts[i] : starts[i] + n])
    one = torch.randn(300, generator=g, device="cuda")
    grads = [one[: t.numel()] for t in lists[0]]
    apart = [[t.clone() for t in ts] for ts in lists]
    tb.adamw_step(lists[0], grads, lists[1], lists[2], step=3, lr=0.1)
    tb.adamw_step(apart[0], [t.clone() for t in grads], apart[1], apart[2], step=3, lr=0.1)
    for a, b in zip(parts(*lists), parts(*apart)):
        assert torch.equal(a, b)


def test_empty_tensors_are_nowhere():
    p, g, m, v = fresh(32)
    none = p[0][:0]
    tb.adamw_step([p[0], none, none], [g[0], none, none], [m[0], none, none], [v[0], none, none], step=1, lr=0.1)
