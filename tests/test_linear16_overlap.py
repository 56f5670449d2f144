"""nllb_linear16 refuses an out that shares memory with what it reads; the addresses are never followed."""
import ctypes

import pytest

import nllb_attn as na

P = 1 << 30


def args(**kw):
    # x: 100 rows of 64 at P, w: 40 rows, out and residual: 100 rows of 40
    a = dict(x=P, w=P + (1 << 20), bias=P + (2 << 20), residual=P + (3 << 20), out=P + (4 << 20), ldx=64, ldw=64, ldr=40, ldo=40,
             dtype=na.BF16, out_dtype=na.BF16, act=0, M=100, N=40, K=64)
    a.update(kw)
    return na.Linear16Args(**a)


OUT = P + (4 << 20)


@pytest.mark.parametrize("kw,needle", [
    (dict(out=P), "x, w or bias"),
    (dict(out=P + 100 * 128 - 2), "x, w or bias"),              # the last value of x
    (dict(out=P - 100 * 80 + 2), "x, w or bias"),               # the first one
    (dict(out=P + (1 << 20) + 40 * 128 - 2), "x, w or bias"),   # of w
    (dict(out=P + (2 << 20) + 78), "x, w or bias"),             # of bias
    (dict(x=OUT + 64, ldx=128, ldo=128), "x, w or bias"),       # columns 32..95 of a matrix whose columns 0..39 are out
    (dict(x=OUT - 96, ldx=128, ldo=128), "x, w or bias"),
    (dict(x=OUT - 112 - 256 * 99, ldx=128, ldo=128), "x, w or bias"),  # (its last row)
    (dict(x=OUT + 80, ldx=128, ldo=120), "x, w or bias"),       # rows that drift into one another
    (dict(residual=OUT, ldr=48), "residual"),                   # the same start, other rows
    (dict(residual=OUT + 2), "residual"),
    (dict(residual=OUT - 80), "residual"),
    (dict(residual=OUT + 80 * 99), "residual"),
    (dict(out_dtype=na.F32, residual=OUT + 4), "residual"),
    (dict(M=1, residual=OUT + 2), "residual"),
])
def test_refuses(kw, needle):
    lib = na.load()
    assert lib.nllb_linear16(ctypes.byref(args(**kw)), None) == na.EINVAL
    assert needle in lib.nllb_attn_last_error().decode()
    assert lib.nllb_linear16_reporting(ctypes.byref(args(**kw)), P, None) == na.EINVAL
