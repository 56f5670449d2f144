"""A launch of nllb_linear16 that gives up with stages still asked for, or with none left to ask for, leaves the GPU and its
next launches as they were."""
import pytest
import torch

import nllb_attn as na

pytestmark = pytest.mark.gpu


# Stages of k of each form's first tile: fewer than a CTA holds at a time (all are asked for before it gives up), and more.
@pytest.mark.parametrize("M,N,K", [(60, 200, 1088), (60, 1000, 2048), (30, 60, 33000), (20000, 100, 64), (30000, 100, 2000),
                                   (300, 20000, 64), (4096, 8192, 1088), (4096, 8192, 128)])
@pytest.mark.parametrize("wide", [False, True], ids=["same", "wide"])
def test_next_launches(cuda_device, M, N, K, wide):
    g = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randint(-2, 3, (M, -(-K // 8) * 8), generator=g, device="cuda").to(torch.float16)[:, :K]
    w = torch.randint(-1, 2, (N, -(-K // 8) * 8), generator=g, device="cuda").to(torch.float16)[:, :K]
    r = torch.ones(M, N, dtype=torch.float32 if wide else torch.float16, device="cuda")
    some = torch.randint(0, M, (50,), generator=g, device="cuda")
    want = (x[some].double() @ w.double().T + 1).to(r.dtype)  # (whole numbers below 2^24: exact in fp32)
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    outs = []
    for i in range(6):
        out = torch.full_like(r, 7.0)
        if i % 2 == 0:
            na.linear16_test_expire_next_wait()
        na.linear16(x, w, residual=r, out=out, error=word)
        outs.append(out)
    torch.cuda.synchronize()
    assert int(word) != 0
    for i, out in enumerate(outs):
        assert (out == 7.0).all() if i % 2 == 0 else torch.equal(out[some], want)
    assert na.linear16_status() == na.OK
