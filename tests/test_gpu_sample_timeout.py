"""The bounded wait of nllb_sample runs out: the rows say so, distinctly from unusable rows, and the next call is exact."""
import pytest
import torch

import nllb_attn as na
from test_gpu_sample import check, f32, i32, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,ld", [(1, 1000, 1000), (200, 3001, 3008), (3, 100003, 100008), (2, 100003, 100003)],
                         ids=["cta", "ctas", "clusters", "unaligned"])
def test_wait_runs_out(cuda_device, rows, vocab, ld, dtype):
    lg, u = make(rows, vocab, dtype, seed=rows, ld=ld)
    k, p = i32([50] * rows), f32([0.9] * rows)
    na.sample_test_expire_next_wait()
    tok, logp = na.sample(lg, u, top_k=k, top_p=p)
    torch.cuda.synchronize()
    assert (tok == na.SAMPLE_TIMEOUT).all() and torch.isneginf(logp).all()
    tok, logp = na.sample(lg, u, top_k=k, top_p=p)
    torch.cuda.synchronize()
    check(lg, u, tok, logp, None, k, p, None, "after the timeout")
    bad, _ = na.sample(torch.full_like(lg, -float("inf")), u)
    assert (bad == -1).all()
