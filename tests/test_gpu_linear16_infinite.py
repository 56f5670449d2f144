"""nllb_linear16's activations where a sum is infinite: what their definitions give in the limit, exactly."""
import math

import pytest
import torch

import nllb_attn as na

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan
# of +inf, -inf, NaN and a large number (of which nothing is taken away)
LIMITS = {"none": (INF, -INF, NAN, 2.0 ** 15), "relu": (INF, 0.0, NAN, 2.0 ** 15), "gelu": (INF, 0.0, NAN, 2.0 ** 15),
          "gelu_tanh": (INF, 0.0, NAN, 2.0 ** 15), "silu": (INF, 0.0, NAN, 2.0 ** 15)}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("wide", [False, True], ids=["same", "wide"])
@pytest.mark.parametrize("act", list(na.ACTIVATIONS))
@pytest.mark.parametrize("M,N,K", [(4, 200, 256), (50, 200, 1024), (60, 1000, 2048), (300, 20000, 64), (4096, 8192, 128),
                                   (30000, 100, 64), (1000, 1024, 4096)])
def test_limits(cuda_device, M, N, K, act, wide, dtype):
    """On each of the forms: few rows, and blocks of them, a cluster per tile, single CTAs, pairs; by a row of x and by the bias,
    each of which decides the whole sum, and with a finite residual behind."""
    x, w = torch.zeros(M, K, dtype=dtype, device="cuda"), torch.zeros(N, K, dtype=dtype, device="cuda")
    w[:, 3] = 1
    given = (INF, -INF, NAN, 2.0 ** 15)
    want = torch.zeros(M, N, dtype=torch.float32, device="cuda")
    bias = torch.zeros(N, dtype=dtype, device="cuda")
    for i, (a, b) in enumerate(zip(given, LIMITS[act])):
        row, col = (M - 1) * (i + 1) // 4, (N - 1) * (i + 1) // 4
        x[row, 3], want[row] = a, b
        bias[col] = a
    for i, b in enumerate(LIMITS[act]):
        col = (N - 1) * (i + 1) // 4
        rows = torch.ones(M, dtype=torch.bool, device="cuda")
        for j in range(4):
            rows[(M - 1) * (j + 1) // 4] = False
        want[rows, col] = b
    crossing = torch.zeros(M, N, dtype=torch.bool, device="cuda")  # (two of the values meet there)
    crossing[[(M - 1) * (i + 1) // 4 for i in range(4)]] = True
    columns = torch.zeros(N, dtype=torch.bool, device="cuda")
    columns[[(N - 1) * (i + 1) // 4 for i in range(4)]] = True
    crossing &= columns
    kind = torch.float32 if wide else dtype
    for residual in (None, torch.ones(M, N, dtype=kind, device="cuda")):
        out = na.linear16(x, w, bias, residual, act, out_dtype=kind)
        ref = (want if residual is None else want + 1).to(kind)
        assert torch.equal(torch.isnan(out)[~crossing], torch.isnan(ref)[~crossing])
        here = ~crossing & ~torch.isnan(ref)
        assert torch.equal(out[here], ref[here])
    assert na.linear16_status() == na.OK
