"""Refusals of the AdamW entry point, and its hash: host code, no GPU."""

import ctypes

import numpy as np
import pytest
import torch

from thingy_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def ptrs(*values):
    return (ctypes.c_void_p * len(values))(*values)


def call(lib, p=256, g=256, m=256, v=256, n=10, p_dtype=_lib.DTYPE_F32, g_dtype=_lib.DTYPE_F32, ms=None, vs=None, step=1,
         step_ptr=None, lr=0.1, lr_ptr=None, b1=0.9, b2=0.99, eps=1e-8, decay=0.0, clip=None, count=1):
    one = lambda x: None if x is None else ptrs(*([x] * max(count, 1)))  # noqa: E731
    sizes = (ctypes.c_int64 * max(count, 1))(*([n] * max(count, 1)))
    return lib.cutie_adamw(count, ptrs(p), p_dtype, ptrs(g), g_dtype, ptrs(m), one(ms), ptrs(v), one(vs), sizes, step, step_ptr, lr,
                           lr_ptr, b1, b2, eps, decay, clip, 0, None)


@pytest.mark.parametrize("kw,status", [
    (dict(count=-1), _lib.ERR_INVALID_ARGUMENT), (dict(p_dtype=7), _lib.ERR_INVALID_ARGUMENT),
    (dict(g_dtype=7), _lib.ERR_INVALID_ARGUMENT), (dict(g_dtype=_lib.DTYPE_F16), _lib.ERR_UNSUPPORTED),
    (dict(p_dtype=_lib.DTYPE_F16, g_dtype=_lib.DTYPE_BF16), _lib.ERR_UNSUPPORTED),
    (dict(b1=1.0), _lib.ERR_INVALID_ARGUMENT), (dict(b2=float("nan")), _lib.ERR_INVALID_ARGUMENT),
    (dict(b1=-0.1), _lib.ERR_INVALID_ARGUMENT), (dict(eps=-1.0), _lib.ERR_INVALID_ARGUMENT),
    (dict(decay=float("nan")), _lib.ERR_INVALID_ARGUMENT), (dict(lr=float("inf")), _lib.ERR_INVALID_ARGUMENT),
    (dict(step=0), _lib.ERR_INVALID_ARGUMENT), (dict(step_ptr=12), _lib.ERR_ALIGNMENT), (dict(lr_ptr=2), _lib.ERR_ALIGNMENT),
    (dict(clip=1), _lib.ERR_ALIGNMENT), (dict(ms=256), _lib.ERR_INVALID_ARGUMENT), (dict(n=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(p=None), _lib.ERR_INVALID_ARGUMENT), (dict(v=None), _lib.ERR_INVALID_ARGUMENT), (dict(p=258), _lib.ERR_ALIGNMENT),
    (dict(m=257), _lib.ERR_ALIGNMENT), (dict(ms=257, vs=256, m=257), _lib.ERR_ALIGNMENT), (dict(count=0), _lib.OK),
    (dict(count=1, n=0, p=None), _lib.OK),
])
def test_refusals(lib, kw, status):
    assert call(lib, **kw) == status


def test_hash_bits_are_even():
    """Each of the 32 bits is set in half of the elements, for neighbours and for strides (six deviations)."""
    mask = 0xFFFFFFFF

    def mix(x):
        x = x ^ (x >> 16)
        x = (x * 0x9E3779B9) & mask
        x = x ^ (x >> 15)
        x = (x * 0x6A09E667) & mask
        return x ^ (x >> 16)

    n = 1 << 16
    for start, stride in ((0, 1), (12345, 128), (7, 4096)):
        for key in (0, 1, 0xDEADBEEF):
            h = mix(((start + stride * torch.arange(n)) * 0x9E3779B9 + key) & mask)
            ones = torch.stack([(h >> b & 1).double().mean() for b in range(32)])
            assert bool(((ones - 0.5).abs() <= 6 * 0.5 / n**0.5).all())
            pair = (h & 0xFFFF).double() / 65536 - 0.5, (h >> 16).double() / 65536 - 0.5
            # the two halves of a hash, and neighbours', are not alike: a mean product of n uniform pairs
            for a, b in (pair, (pair[0][1:], pair[0][:-1])):
                assert abs(float((a * b).mean())) <= 6 / 12 / n**0.5


def test_square_root_iteration_is_correctly_rounded():
    """Markstein's iteration as the kernel makes it, from every start within two ulps, for every mantissa of two
    binades (a power of four changes exponents alone). Products of fp32 values are exact in 64 bits, and so are the
    residuals; the last sum is rounded by its exact correction in ulps."""
    f32, f64 = np.float32, np.float64
    for base in (0x3F800000, 0x40000000):
        for at in range(0, 1 << 23, 1 << 21):
            a = np.arange(base + at, base + at + (1 << 21), dtype=np.uint32).view(f32).astype(f64)
            s = np.sqrt(a)  # 53 bits: a root is never so near to the middle of two fp32 values
            want = s.astype(f32)
            for k in (-2, -1, 0, 1, 2):
                y = ((1.0 / s).astype(f32).view(np.int32) + np.int32(k)).view(f32).astype(f64)
                g, h = (a * y).astype(f32).astype(f64), 0.5 * y
                r = (0.5 - g * h).astype(f32).astype(f64)
                g1, h1 = (g + g * r).astype(f32), (h + h * r).astype(f32).astype(f64)
                d = (a - g1.astype(f64) ** 2).astype(f32).astype(f64)
                ulp = np.spacing(g1).astype(f64)
                got = (g1.astype(f64) + np.rint(d * h1 / ulp) * ulp).astype(f32)
                assert np.array_equal(got, want)
