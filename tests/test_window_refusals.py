"""What nllb_attn_window refuses before touching a GPU."""
import ctypes

import pytest

import nllb_attn as na
from test_rows_sample_refusals import paged_args


def status(window=5, sinks=1, **kw):
    lib = na.load()
    rc = lib.nllb_attn_window(None, ctypes.byref(na.WindowArgs(paged_args(**kw), window, sinks)))
    return rc, lib.nllb_attn_last_error().decode()


@pytest.mark.parametrize("kw,code,needle", [
    (dict(window=0), na.EINVAL, "window"),
    (dict(window=-3), na.EINVAL, "window"),
    (dict(sinks=-1), na.EINVAL, "sinks"),
    (dict(dtype=3), na.EINVAL, "dtype"),
    (dict(head_dim=32), na.EINVAL, "head_dim"),
    (dict(n_seq=70000), na.ECAPACITY, "sequences"),
    (dict(scale=float("inf")), na.EINVAL, "scale"),
    (dict(page_table=None), na.EINVAL, "required"),
    (dict(max_kv=65), na.EINVAL, "page_table_stride"),
    (dict(q_rows=3), na.EINVAL, "q_rows"),
    (dict(out_stride_row=0), na.EINVAL, "overlap"),
])
def test_refuses(kw, code, needle):
    rc, text = status(**kw)
    assert rc == code and needle in text


def test_valid_arguments_still_need_a_context():
    for kw in (dict(), dict(window=2 ** 31 - 1, sinks=2 ** 31 - 1), dict(n_seq=0)):
        rc, text = status(**kw)
        assert rc == na.EINVAL and "ctx" in text
    assert na.load().nllb_attn_window(None, None) == na.EINVAL
