"""Refusals of the experts' products and of the sorted cast: host code, no GPU."""

import pytest

from thingy_b200 import _lib

FAKE = 1 << 20  # an aligned address that no refused call reaches


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def gemm(lib, **kw):
    args = dict(a=FAKE, lda=512, a_scale=FAKE, sa_row=4, sa_kb=1, b=FAKE, ldb=512, b_expert=256 * 512, b_scale=FAKE, sb_row=4, sb_kb=1,
                sb_expert=8, offsets=FAKE, counts=FAKE, E=8, d=FAKE, ldd=256, d_dtype=_lib.DTYPE_BF16, R=1024, N=256, K=512, stream=None)
    assert set(kw) <= set(args)
    return lib.cutie_fp8_grouped_gemm(*{**args, **kw}.values())


def wgrad(lib, **kw):
    args = dict(a=FAKE, lda=1024, a_scale=FAKE, sa_row=1, sa_kb=256, b=FAKE, ldb=1024, b_scale=FAKE, sb_row=1, sb_kb=512, offsets=FAKE,
                E=8, d=FAKE, ldd=512, d_expert=256 * 512, d_dtype=_lib.DTYPE_F32, R=1024, N=256, K=512, stream=None)
    assert set(kw) <= set(args)
    return lib.cutie_fp8_grouped_wgrad(*{**args, **kw}.values())


def cast(lib, **kw):
    args = dict(x=FAKE, ldx=256, R=1024, H=256, sources=FAKE, scale_fmt=_lib.SCALE_FP32, q=FAKE, ldq=256, s=FAKE, lds=1024, qt=FAKE,
                ldqt=1024, st=FAKE, ldst=256, stream=None)
    assert set(kw) <= set(args)
    return lib.cutie_cast_fp8_sorted(*{**args, **kw}.values())


COMMON = [
    ({"E": 0}, _lib.ERR_INVALID_ARGUMENT), ({"E": 513}, _lib.ERR_UNSUPPORTED), ({"R": -128}, _lib.ERR_INVALID_ARGUMENT),
    ({"R": 1000}, _lib.ERR_UNSUPPORTED), ({"R": 2**31}, _lib.ERR_UNSUPPORTED), ({"N": 0}, _lib.ERR_INVALID_ARGUMENT),
    ({"K": 0}, _lib.ERR_INVALID_ARGUMENT), ({"N": 2**25}, _lib.ERR_UNSUPPORTED), ({"d_dtype": _lib.DTYPE_F16}, _lib.ERR_INVALID_ARGUMENT),
    ({"offsets": None}, _lib.ERR_INVALID_ARGUMENT), ({"offsets": FAKE + 2}, _lib.ERR_ALIGNMENT), ({"a": None}, _lib.ERR_INVALID_ARGUMENT),
    ({"a": FAKE + 8}, _lib.ERR_ALIGNMENT), ({"b": FAKE + 8}, _lib.ERR_ALIGNMENT), ({"a_scale": None}, _lib.ERR_INVALID_ARGUMENT),
    ({"b_scale": FAKE + 1}, _lib.ERR_ALIGNMENT), ({"sa_row": -1}, _lib.ERR_INVALID_ARGUMENT), ({"d": None}, _lib.ERR_INVALID_ARGUMENT),
    ({"d": FAKE + 16}, _lib.ERR_ALIGNMENT), ({"lda": 100}, _lib.ERR_INVALID_ARGUMENT), ({"ldd": 128}, _lib.ERR_INVALID_ARGUMENT),
]


@pytest.mark.parametrize("kw,status", COMMON + [
    ({"counts": FAKE + 1}, _lib.ERR_ALIGNMENT), ({"b_expert": 8}, _lib.ERR_ALIGNMENT), ({"sb_expert": -1}, _lib.ERR_ALIGNMENT),
    ({"N": 248}, _lib.ERR_UNSUPPORTED), ({"ldd": 264}, _lib.ERR_ALIGNMENT), ({"R": 0}, _lib.OK),
])
def test_product(lib, kw, status):
    assert gemm(lib, **kw) == status
    if status != _lib.OK:
        assert lib.cutie_last_error() != b""


@pytest.mark.parametrize("kw,status", COMMON + [
    ({"d_expert": 4}, _lib.ERR_ALIGNMENT), ({"d_expert": -8}, _lib.ERR_ALIGNMENT), ({"K": 508}, _lib.ERR_UNSUPPORTED),
    ({"ldd": 516}, _lib.ERR_ALIGNMENT), ({"lda": 1032}, _lib.ERR_ALIGNMENT),
])
def test_weight_gradient(lib, kw, status):
    assert wgrad(lib, **kw) == status


@pytest.mark.parametrize("kw,status", [
    ({"R": 100}, _lib.ERR_UNSUPPORTED), ({"sources": None}, _lib.ERR_INVALID_ARGUMENT), ({"sources": FAKE + 2}, _lib.ERR_ALIGNMENT),
    ({"x": FAKE + 2}, _lib.ERR_ALIGNMENT), ({"ldx": 248}, _lib.ERR_INVALID_ARGUMENT), ({"H": 4}, _lib.ERR_UNSUPPORTED),
    ({"qt": None, "st": None}, _lib.ERR_INVALID_ARGUMENT), ({"R": 0}, _lib.OK),
])
def test_sorted_cast(lib, kw, status):
    assert cast(lib, **kw) == status
