"""The gradient form of the tile cast at its C entry point: what it refuses, before touching CUDA."""

import ctypes

import pytest

from thingy_b200 import _lib
from test_block_capi import FAKE, _refused, cast, lib  # noqa: F401

POW2 = _lib.SCALE_FP32_POW2


@pytest.mark.parametrize("kw,code,needle", [
    ({"scale_fmt": _lib.SCALE_GRADIENT, "tile_kind": _lib.TILE_BLOCK}, _lib.ERR_UNSUPPORTED, "two-way"),
    ({"scale_fmt": _lib.SCALE_GRADIENT + POW2, "tile_kind": _lib.TILE_BLOCK}, _lib.ERR_UNSUPPORTED, "two-way"),
    ({"scale_fmt": _lib.SCALE_GRADIENT + _lib.SCALE_E8M0}, _lib.ERR_UNSUPPORTED, "fp32 scales"),
    ({"scale_fmt": 2 * _lib.SCALE_GRADIENT}, _lib.ERR_UNSUPPORTED, "fp32 scales"),
    ({"scale_fmt": _lib.SCALE_GRADIENT, "qt": None, "st": None}, _lib.ERR_INVALID_ARGUMENT, "two-way"),
    ({"scale_fmt": _lib.SCALE_GRADIENT, "x": ctypes.c_void_p(0x10001)}, _lib.ERR_ALIGNMENT, "x: rows"),
])
def test_gradient_cast_refusals(lib, kw, code, needle):  # noqa: F811
    _refused(lib, cast(lib, **kw), code, needle)


@pytest.mark.parametrize("fmt", [_lib.SCALE_GRADIENT, _lib.SCALE_GRADIENT + POW2])
def test_gradient_cast_of_no_rows_needs_no_gpu(lib, fmt):  # noqa: F811
    assert cast(lib, M=0, scale_fmt=fmt, x=FAKE) == _lib.OK
