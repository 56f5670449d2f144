"""What nllb_logprobs refuses before touching a GPU."""
import ctypes

import pytest

import nllb_attn as na

P = 1 << 20  # an address that is never followed


def args(**kw):
    a = dict(logits=P, ld=100, dtype=na.F32, vocab=100, rows=2, top_n=3, target=P, out_logp=P, out_entropy=P, out_top_tok=P,
             out_top_logp=P)
    a.update(kw)
    return na.LogprobsArgs(**a)


@pytest.mark.parametrize("kw,status,needle", [
    (dict(dtype=3), na.EINVAL, "dtype"),
    (dict(rows=-1), na.EINVAL, "rows"),
    (dict(vocab=0), na.EINVAL, "vocab"),
    (dict(vocab=2 ** 30 + 1, ld=2 ** 31), na.ECAPACITY, "logits"),
    (dict(rows=2 ** 26 + 1), na.ECAPACITY, "logits"),
    (dict(top_n=-1), na.EINVAL, "top_n"),
    (dict(top_n=33), na.ECAPACITY, "top_n"),
    (dict(logits=None), na.EINVAL, "logits"),
    (dict(target=None), na.EINVAL, "target"),
    (dict(out_top_tok=None), na.EINVAL, "top_n"),
    (dict(out_top_logp=None), na.EINVAL, "top_n"),
    (dict(out_logp=None, out_entropy=None, top_n=0), na.EINVAL, "output"),
    (dict(ld=99), na.EINVAL, "ld"),
    (dict(logits=P + 2), na.EINVAL, "aligned"),
    (dict(logits=P + 1, dtype=na.BF16), na.EINVAL, "aligned"),
])
def test_refuses(kw, status, needle):
    lib = na.load()
    assert lib.nllb_logprobs(ctypes.byref(args(**kw)), None) == status
    assert needle in lib.nllb_attn_last_error().decode()


def test_no_rows_is_nothing():
    lib = na.load()
    assert lib.nllb_logprobs(ctypes.byref(args(rows=0, logits=None)), None) == na.OK
    assert lib.nllb_logprobs(None, None) == na.EINVAL


def test_binding_checks_tensors():
    import torch
    x, t = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int32)
    for args_, kw in [((x.t(),), {}), ((x, t), {}), ((x,), dict(out_logp=torch.zeros(4))), ((x,), dict(top_n=33)),
                      ((x,), dict(top_n=-1))]:
        with pytest.raises(ValueError):
            na.logprobs(*args_, **kw)
