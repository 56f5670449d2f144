"""What nllb_linear16_reporting refuses before touching a GPU."""
import ctypes

import pytest

import nllb_attn as na
from test_linear16_refusals import P, args


@pytest.mark.parametrize("error,kw,needle", [(None, {}, "error"), (P + 2, {}, "aligned"), (P, dict(K=0), "K"),
                                             (P, dict(ldx=56), "ldx")])
def test_refuses(error, kw, needle):
    lib = na.load()
    assert lib.nllb_linear16_reporting(ctypes.byref(args(**kw)), error, None) == na.EINVAL
    assert needle in lib.nllb_attn_last_error().decode()


def test_no_rows_is_nothing():
    lib = na.load()
    assert lib.nllb_linear16_reporting(ctypes.byref(args(M=0, x=None)), P, None) == na.OK
    assert lib.nllb_linear16_reporting(None, P, None) == na.EINVAL
