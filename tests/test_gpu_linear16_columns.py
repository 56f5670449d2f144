"""nllb_linear16 into columns of a wider matrix whose rows start on 16 bytes: what lies behind the last column stays."""
import pytest
import torch

import nllb_attn as na
from test_gpu_linear16 import TYPES, check, normal, rows

pytestmark = pytest.mark.gpu


def into_columns(M, N, K, dtype, wide, residual, act="none", behind=8):
    g = torch.Generator(device="cuda").manual_seed(M * 31 + N * 7 + K)
    kind = torch.float32 if wide else dtype
    x, w = rows(g, M, K, dtype), rows(g, N, K, dtype, K ** -0.5)
    b = normal(g, N, dtype=dtype)
    ld = -(-N // 8) * 8 + behind
    whole = normal(g, M, ld, dtype=kind)
    before = whole.clone()
    out = whole[:, :N]
    r = {"none": None, "in place": out, "beside": normal(g, M, ld, dtype=kind)[:, :N], "anywhere": normal(g, M, ld + 1, dtype=kind)[:, :N]}[residual]
    na.linear16(x, w, b, r, act, out)
    torch.cuda.synchronize()
    check(out, x, w, b, before[:, :N] if residual == "in place" else r, act, f"{M} x {N} x {K}")
    assert torch.equal(whole[:, N:], before[:, N:]), f"{M} x {N} x {K}"


@pytest.mark.parametrize("wide", [False, True], ids=["same", "wide"])
@pytest.mark.parametrize("residual", ["none", "in place", "beside", "anywhere"])
@pytest.mark.parametrize("M,K", [(5, 100), (12000, 200), (300, 64), (60, 2048), (4096, 128), (20000, 2000), (1000, 4096)])
def test_every_width(cuda_device, M, K, residual, wide):
    """Few rows, single CTAs, pairs, clusters; each rest of 32 columns and of 16 bytes."""
    for N in list(range(1, 35)) + [63, 97, 127, 129, 250, 1001]:
        into_columns(M, N, K, TYPES[N % 2], wide, residual)


@pytest.mark.parametrize("wide", [False, True], ids=["same", "wide"])
@pytest.mark.parametrize("residual", ["none", "in place", "beside", "anywhere"])
@pytest.mark.parametrize("M,N,K", [(64, 50003, 128), (64, 50003, 1100), (300, 20001, 64), (300, 20030, 1100), (4096, 8191, 128),
                                   (5000, 1030, 500), (700, 40012, 155), (3000, 4099, 200)])
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_tiles_of_both_kinds(cuda_device, M, N, K, residual, act, wide):
    """CTAs that go from tiles within the columns to those of their end, and back."""
    for dtype in TYPES:
        into_columns(M, N, K, dtype, wide, residual, act)


def test_the_end_of_a_buffer(cuda_device):
    """The last row ends where the buffer does: whatever follows there is of others."""
    for M, N, K, kind in ((300, 20001, 64, torch.float16), (4096, 1001, 128, torch.float32), (300, 30, 64, torch.bfloat16)):
        dtype = torch.float16 if kind == torch.float32 else kind
        ld = -(-N // 8) * 8
        flat = torch.full(((M - 1) * ld + N + 64,), 7.0, dtype=kind, device="cuda")
        out = flat[:(M - 1) * ld + N].as_strided((M, N), (ld, 1))
        x, w = torch.ones(M, K, dtype=dtype, device="cuda"), torch.ones(N, K, dtype=dtype, device="cuda")
        na.linear16(x, w, out=out)
        torch.cuda.synchronize()
        assert (out == K).all() and (flat[(M - 1) * ld + N:] == 7.0).all()
