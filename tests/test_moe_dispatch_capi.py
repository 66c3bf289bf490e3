"""Sizes and refusals of the sort and row entry points: host code, no GPU."""

import pytest

from thingy_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.mark.parametrize("T,k,E,align", [(0, 1, 1, 1), (1, 8, 128, 128), (1, 8, 4, 128), (1000, 3, 8, 16), (5, 2, 512, 65536)])
def test_plan_rows(lib, T, k, E, align):
    n = T * k
    assert lib.cutie_moe_plan_rows(T, k, E, align) == (n + min(E, n) * (align - 1)) // align * align


@pytest.mark.parametrize("sizes", [(-1, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 513, 1), (1, 1, 1, 0), (1, 1, 1, 65537),
                                   (2**30, 2, 1, 1), (2**31, 1, 1, 1), (2**62, 2**62, 1, 1)])
def test_plan_rows_refused(lib, sizes):
    assert lib.cutie_moe_plan_rows(*sizes) == -1
    assert lib.cutie_last_error() != b""


def test_workspace_only_above_one_cta(lib):
    assert lib.cutie_moe_sort_workspace(512, 8, 64) == 0
    assert lib.cutie_moe_sort_workspace(513, 8, 64) == 3 * 64 * 4
    assert lib.cutie_moe_sort_workspace(2**27, 8, 512) == 128 * 512 * 4


def test_sort_refused(lib):
    def sort(ids=256, T=1024, k=8, E=64, align=128, sources=256, R=None, offsets=256, workspace=256, size=1 << 20):
        R = lib.cutie_moe_plan_rows(T, k, E, align) if R is None else R
        return lib.cutie_moe_sort(ids, 0, T, k, E, align, sources, R, 256, offsets, 256, workspace, size, None)

    assert sort(R=lib.cutie_moe_plan_rows(1024, 8, 64, 128) - 1) == _lib.ERR_INVALID_ARGUMENT
    assert sort(R=2**31) == _lib.ERR_INVALID_ARGUMENT
    assert sort(ids=None) == _lib.ERR_INVALID_ARGUMENT
    assert sort(offsets=None) == _lib.ERR_INVALID_ARGUMENT
    assert sort(sources=258) == _lib.ERR_ALIGNMENT
    assert sort(workspace=None) == _lib.ERR_INVALID_ARGUMENT
    assert sort(size=4 * 64 * 4 - 1) == _lib.ERR_INVALID_ARGUMENT
    assert sort(E=1000, R=8192) == _lib.ERR_UNSUPPORTED


def test_rows_refused(lib):
    def permute(x=256, ldx=64, es=2, T=4, H=64, k=2, positions=256, sources=256, R=8, out=256, ldo=64):
        return lib.cutie_moe_permute(x, ldx, es, T, H, k, positions, sources, R, out, ldo, None)

    assert permute(es=8) == _lib.ERR_UNSUPPORTED
    assert permute(x=None) == _lib.ERR_INVALID_ARGUMENT
    assert permute(x=257) == _lib.ERR_ALIGNMENT
    assert permute(ldx=63) == _lib.ERR_INVALID_ARGUMENT
    assert permute(ldo=63) == _lib.ERR_INVALID_ARGUMENT
    assert permute(out=None) == _lib.ERR_INVALID_ARGUMENT
    assert permute(positions=None) == _lib.ERR_INVALID_ARGUMENT
    assert permute(sources=None) == _lib.ERR_INVALID_ARGUMENT
    assert permute(sources=257) == _lib.ERR_ALIGNMENT
    assert permute(H=0) == _lib.ERR_INVALID_ARGUMENT
    assert permute(R=2**31) == _lib.ERR_UNSUPPORTED
    assert permute(T=2**30, k=2) == _lib.ERR_UNSUPPORTED
    assert permute(T=0, R=0) == _lib.OK  # nothing to do

    def combine(rows=256, dtype=_lib.DTYPE_BF16, weights=256, positions=256, T=4, out=256, ldr=64):
        return lib.cutie_moe_combine(rows, ldr, dtype, weights, positions, T, 2, 64, 8, out, 64, None)

    assert combine(dtype=3) == _lib.ERR_INVALID_ARGUMENT
    assert combine(rows=None) == _lib.ERR_INVALID_ARGUMENT
    assert combine(weights=258) == _lib.ERR_ALIGNMENT
    assert combine(ldr=8) == _lib.ERR_INVALID_ARGUMENT
    assert combine(out=None) == _lib.ERR_INVALID_ARGUMENT
    assert combine(T=0) == _lib.OK

    def backward(dy=256, rows=256, weights=256, drows=256, dw=256, sources=256):
        return lib.cutie_moe_combine_backward(dy, 64, rows, 64, _lib.DTYPE_F32, weights, 256, sources, 4, 2, 64, 8, drows, 64, dw, None)

    assert backward(dy=None) == _lib.ERR_INVALID_ARGUMENT
    assert backward(rows=None) == _lib.ERR_INVALID_ARGUMENT
    assert backward(weights=None) == _lib.ERR_INVALID_ARGUMENT
    assert backward(sources=None) == _lib.ERR_INVALID_ARGUMENT
    assert backward(dw=258) == _lib.ERR_ALIGNMENT
    assert backward(drows=None, dw=None) == _lib.OK
