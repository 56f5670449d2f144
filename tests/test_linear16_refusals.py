"""What nllb_linear16 refuses before touching a GPU."""
import ctypes

import pytest

import nllb_attn as na

P = 1 << 20  # an address that is never followed


def args(**kw):
    a = dict(x=P, w=P, bias=P, residual=P, out=P, ldx=64, ldw=64, ldr=100, ldo=100, dtype=na.BF16, out_dtype=na.BF16, act=1,
             M=3, N=100, K=64)
    a.update(kw)
    return na.Linear16Args(**a)


@pytest.mark.parametrize("kw,status,needle", [
    (dict(dtype=na.F32, out_dtype=na.F32), na.EINVAL, "dtype"),
    (dict(dtype=7), na.EINVAL, "dtype"),
    (dict(out_dtype=na.F16), na.EINVAL, "out_dtype"),
    (dict(act=5), na.EINVAL, "act"),
    (dict(act=-1), na.EINVAL, "act"),
    (dict(M=-1), na.EINVAL, "M"),
    (dict(N=0), na.EINVAL, "N"),
    (dict(K=0), na.EINVAL, "K"),
    (dict(M=2 ** 24 + 1), na.ECAPACITY, "2^24"),
    (dict(M=2 ** 24, N=2 ** 24, ldo=2 ** 24, ldr=2 ** 24), na.ECAPACITY, "outputs"),
    (dict(x=None), na.EINVAL, "required"),
    (dict(w=None), na.EINVAL, "required"),
    (dict(out=None), na.EINVAL, "required"),
    (dict(ldx=56), na.EINVAL, "ldx"),
    (dict(ldw=56), na.EINVAL, "ldw"),
    (dict(ldo=99), na.EINVAL, "ldo"),
    (dict(ldr=99), na.EINVAL, "ldr"),
    (dict(ldx=68), na.EINVAL, "multiples of 8"),
    (dict(w=P + 8), na.EINVAL, "16-byte"),
    (dict(ldw=2 ** 37), na.ECAPACITY, "2^36"),
    (dict(out=P + 1), na.EINVAL, "aligned"),
    (dict(out=P + 2, out_dtype=na.F32), na.EINVAL, "aligned"),
    (dict(bias=P + 1), na.EINVAL, "aligned"),
    (dict(residual=P + 1), na.EINVAL, "aligned"),
])
def test_refuses(kw, status, needle):
    lib = na.load()
    assert lib.nllb_linear16(ctypes.byref(args(**kw)), None) == status
    assert needle in lib.nllb_attn_last_error().decode()


def test_no_rows_is_nothing():
    lib = na.load()
    assert lib.nllb_linear16(ctypes.byref(args(M=0, x=None)), None) == na.OK
    assert lib.nllb_linear16(None, None) == na.EINVAL


def test_binding_checks_tensors():
    import torch
    x, w = torch.zeros(3, 64).half(), torch.zeros(5, 64).half()
    for a, kw in [((x.float(), w.float()), {}), ((x, w), {}), ((x, w), dict(act="tanh")), ((x, w), dict(out_dtype=torch.bfloat16)),
                  ((x, w), dict(out=torch.zeros(3, 5), out_dtype=torch.float16))]:
        with pytest.raises(ValueError):
            na.linear16(*a, **kw)
