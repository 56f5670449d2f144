"""nllb_logprobs where two and sixteen CTAs share a row, and rows whose largest logits lie far out, against 64 bits."""
import math

import pytest
import torch

import nllb_attn as na
from test_gpu_logprobs import TYPES, check, logits_of

pytestmark = pytest.mark.gpu


def run(lg, t, n, rows=None):
    """(checked: `rows` of them)"""
    out = na.logprobs(lg, t, top_n=n)
    torch.cuda.synchronize()
    pick = range(len(lg)) if rows is None else rows
    check(lg[list(pick)], t[list(pick)], [None if x is None else x[list(pick)] for x in out], n)
    return out


@pytest.mark.parametrize("n", [0, 1, 32])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 820000), (1, 820001), (3, 1000003), (2, 3000017)])
def test_sixteen_ctas_to_a_row(cuda_device, rows, vocab, dtype, n):
    lg, t = logits_of(rows, vocab, dtype, vocab)
    run(lg, t, n)
    # the likeliest in every part of the row, one by one and crowded into one
    for at in (torch.arange(40) * (vocab // 40) + 7, vocab - 1 - torch.arange(40) * 3, vocab * 9 // 16 + torch.arange(40) * 2048):
        x = lg.clone()
        x[:, at.cuda()] = (20 + torch.arange(40, device="cuda") % 13).to(dtype)
        x[0, at[3]] = math.nan
        run(x, at[:rows].to(torch.int32).cuda(), n)


@pytest.mark.parametrize("n", [0, 1, 32])
@pytest.mark.parametrize("rows,vocab,dtype", [(100, 200000, torch.float32), (100, 200001, torch.float32), (100, 400003, torch.float16),
                                              (100, 400000, torch.bfloat16)])
def test_two_ctas_to_a_row(cuda_device, rows, vocab, dtype, n):
    lg, t = logits_of(rows, vocab, dtype, vocab)
    t[5] = -1
    first = run(lg, t, n, rows=(0, 1, 5, 50, 98, 99))
    again = na.logprobs(lg, t, top_n=n)
    assert all(torch.equal(a, b) for a, b in zip(first, again) if a is not None)


@pytest.mark.parametrize("vocab", [200001, 820001])
@pytest.mark.parametrize("top,step", [(1.2e8, 8), (1.9e8, 16), (2.0e8, 16), (2.6e8, 16), (2.7e8, 32), (-2.0e8, 16)])
def test_far_rows_with_many_tokens_one_step_below(cuda_device, vocab, top, step):
    """Steps of fp32 there: e^-16 each, of 200000 tokens, is 0.02."""
    lg = torch.full((1, vocab), float(top), device="cuda")
    lg[0, 7] = top + step
    assert float(lg[0, 7]) - float(lg[0, 8]) == step
    t = torch.tensor([7], dtype=torch.int32, device="cuda")
    run(lg, t, 2)
