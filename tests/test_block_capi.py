"""The C entry points of the casts, the block-scaled product and the mixture-of-experts
layer reject bad arguments with status codes before touching CUDA (no GPU needed)."""

import ctypes

import pytest

from thingy_b200 import _lib

FAKE = ctypes.c_void_p(0x10000)  # never dereferenced: every call below fails validation
ODD = ctypes.c_void_p(0x10001)


@pytest.fixture(scope="module")
def lib():
    if not _lib.library_path().exists():
        from thingy_b200.build import build

        build()
    return _lib.load()


def _refused(lib, status, code, needle):
    assert status == code
    assert needle in lib.cutie_last_error().decode()


def cast(lib, **kw):
    args = dict(x=FAKE, ldx=256, M=100, H=256, tile_kind=_lib.TILE_TWO_WAY, scale_fmt=0, q=FAKE, ldq=256, s=FAKE,
                lds=100, qt=FAKE, ldqt=112, st=FAKE, ldst=256, stream=None)
    args.update(kw)
    return lib.cutie_cast_fp8_tiles(*args.values())


@pytest.mark.parametrize("kw,code,needle", [
    ({"M": -1}, _lib.ERR_INVALID_ARGUMENT, "M >= 0"),
    ({"H": 0}, _lib.ERR_INVALID_ARGUMENT, "H > 0"),
    ({"H": 252}, _lib.ERR_UNSUPPORTED, "multiple of 8"),
    ({"tile_kind": 2}, _lib.ERR_INVALID_ARGUMENT, "tile_kind"),
    ({"scale_fmt": _lib.SCALE_E8M0}, _lib.ERR_UNSUPPORTED, "fp32 scales"),
    ({"qt": None}, _lib.ERR_INVALID_ARGUMENT, "together"),
    ({"qt": None, "st": None}, _lib.ERR_INVALID_ARGUMENT, "two-way"),
    ({"x": None}, _lib.ERR_INVALID_ARGUMENT, "x is NULL"),
    ({"x": ODD}, _lib.ERR_ALIGNMENT, "x: rows"),
    ({"ldx": 248}, _lib.ERR_INVALID_ARGUMENT, "leading dimension"),
    ({"ldx": 260}, _lib.ERR_ALIGNMENT, "x: rows"),
    ({"ldq": 252 + 8}, _lib.ERR_ALIGNMENT, "q: rows"),
    ({"lds": 99}, _lib.ERR_INVALID_ARGUMENT, "s: leading dimension"),
    ({"ldqt": 96}, _lib.ERR_INVALID_ARGUMENT, "qt: leading dimension"),
    ({"ldst": 128}, _lib.ERR_INVALID_ARGUMENT, "st: leading dimension"),
    ({"tile_kind": _lib.TILE_BLOCK, "lds": 1}, _lib.ERR_INVALID_ARGUMENT, "s: leading dimension"),
    ({"M": 2**40}, _lib.ERR_UNSUPPORTED, "tiles"),
])
def test_cast_refusals(lib, kw, code, needle):
    _refused(lib, cast(lib, **kw), code, needle)


def test_cast_of_no_rows_needs_no_gpu(lib):
    assert cast(lib, M=0) == _lib.OK


def gemm(lib, **kw):
    args = dict(a=FAKE, lda=512, a_scale=FAKE, sa_row=4, sa_kb=1, b=FAKE, ldb=512, b_scale=FAKE, sb_row=4, sb_kb=1,
                b_rows=0, d=FAKE, ldd=256, d_dtype=_lib.DTYPE_BF16, accumulate=0, M=64, N=256, K=512, stream=None)
    args.update(kw)
    return lib.cutie_fp8_block_gemm(*args.values())


@pytest.mark.parametrize("kw,code,needle", [
    ({"M": -1}, _lib.ERR_INVALID_ARGUMENT, ">= 0"),
    ({"N": 2**31}, _lib.ERR_UNSUPPORTED, "below 2^31"),
    ({"d_dtype": 2}, _lib.ERR_INVALID_ARGUMENT, "d_dtype"),
    ({"accumulate": 1}, _lib.ERR_UNSUPPORTED, "fp32 output"),
    ({"d": None}, _lib.ERR_INVALID_ARGUMENT, "d is NULL"),
    ({"ldd": 255}, _lib.ERR_INVALID_ARGUMENT, "leading dimension"),
    ({"d": ODD}, _lib.ERR_ALIGNMENT, "d: rows"),
    ({"a": None}, _lib.ERR_INVALID_ARGUMENT, "a is NULL"),
    ({"lda": 520}, _lib.ERR_ALIGNMENT, "a: rows"),
    ({"ldb": 496}, _lib.ERR_INVALID_ARGUMENT, "leading dimension"),
    ({"b": ODD}, _lib.ERR_ALIGNMENT, "b: rows"),
    ({"a_scale": None}, _lib.ERR_INVALID_ARGUMENT, "scale"),
    ({"b_scale": ODD}, _lib.ERR_ALIGNMENT, "4-byte"),
    ({"sa_kb": -1}, _lib.ERR_INVALID_ARGUMENT, "negative"),
])
def test_product_refusals(lib, kw, code, needle):
    _refused(lib, gemm(lib, **kw), code, needle)


def test_empty_products_need_no_gpu(lib):
    assert gemm(lib, M=0) == _lib.OK
    assert gemm(lib, N=0) == _lib.OK
    assert gemm(lib, K=0, d_dtype=_lib.DTYPE_F32, accumulate=1) == _lib.OK


def moe(lib, **kw):
    args = dict(x=FAKE, ldx=256, q=FAKE, ldq=256, q_scale=FAKE, sq_row=2, sq_kb=1, router=FAKE, bias=None, w13=FAKE,
                w13_scale=FAKE, w2=FAKE, w2_scale=FAKE, T=4, E=8, top_k=2, H=256, I=128, scoring=0, renormalize=1,
                routed_scale=1.0, out=FAKE, ldo=256, topk_ids=None, topk_weights=None, workspace=FAKE,
                workspace_bytes=0, stream=None)
    args.update(kw)
    return lib.cutie_moe_fp8(*args.values())


@pytest.mark.parametrize("kw,code,needle", [
    ({"T": -1}, _lib.ERR_INVALID_ARGUMENT, "T >= 0"),
    ({"T": 65}, _lib.ERR_UNSUPPORTED, "at most 64"),
    ({"E": 513}, _lib.ERR_UNSUPPORTED, "experts"),
    ({"top_k": 9}, _lib.ERR_UNSUPPORTED, "top_k"),
    ({"top_k": 17, "E": 32}, _lib.ERR_UNSUPPORTED, "top_k"),
    ({"H": 192}, _lib.ERR_UNSUPPORTED, "multiples of 128"),
    ({"I": 100}, _lib.ERR_UNSUPPORTED, "multiples of 128"),
    ({"I": 2**20, "E": 512}, _lib.ERR_UNSUPPORTED, "too large"),
    ({"scoring": 2}, _lib.ERR_INVALID_ARGUMENT, "scoring"),
    ({"x": ODD}, _lib.ERR_ALIGNMENT, "x: rows"),
    ({"ldq": 264}, _lib.ERR_ALIGNMENT, "q: rows"),
    ({"w2": None}, _lib.ERR_INVALID_ARGUMENT, "w2 is NULL"),
    ({"w13_scale": None}, _lib.ERR_INVALID_ARGUMENT, "w13_scale"),
    ({"bias": ODD}, _lib.ERR_ALIGNMENT, "4-byte"),
    ({"sq_row": -2}, _lib.ERR_INVALID_ARGUMENT, "negative"),
    ({}, _lib.ERR_INVALID_ARGUMENT, "workspace"),
])
def test_moe_refusals(lib, kw, code, needle):
    _refused(lib, moe(lib, **kw), code, needle)


def test_moe_sizes(lib):
    assert moe(lib, T=0) == _lib.OK
    assert lib.cutie_moe_fp8_workspace(4, 8, 2, 256, 128) > 0
    assert lib.cutie_moe_fp8_workspace(65, 8, 2, 256, 128) == 0
    assert b"at most 64" in lib.cutie_last_error()
