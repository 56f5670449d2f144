"""nllb_linear16 where a sum is taken in several parts, on each of its forms with every epilogue, against 64 bits (tolerances
as in test_gpu_linear16)."""
import pytest
import torch

import nllb_attn as na
from test_gpu_linear16 import TYPES, U, case, check, half_step, normal, rows

pytestmark = pytest.mark.gpu

# sums of more than 1024 (fp32 outputs) or 16384 (16-bit ones) of one CTA, by form
PARTS = [
    # single CTAs
    (20000, 100, 2000, True), (30000, 100, 1100, True), (9500, 128, 1500, True), (4578, 18, 1447, True), (20097, 20, 5462, True),
    (11961, 17, 18058, False), (9242, 17, 35834, False), (14598, 126, 17343, True),
    # pairs
    (2302, 21, 1208, True), (25, 10887, 1746, True), (2100, 4000, 2500, True), (9500, 17, 18959, False), (17, 12135, 35817, False),
    # clusters of two, four and eight that share k
    (2177, 16, 3450, True), (1000, 1024, 4096, True), (19, 4465, 34564, False),
    (300, 1000, 6000, True), (640, 512, 5000, True), (46, 3531, 7802, True), (1916, 16, 11659, True), (200, 1000, 8000, True),
    (18, 16, 8965, True), (1402, 20, 11026, True), (193, 496, 37208, True),
]


def padded(M, N, K, dtype, act, bias, residual, wide, aligned):
    """case(), whose outputs and residual start on 16 bytes row by row where `aligned` says so."""
    if not aligned:
        return case(M, N, K, dtype, act, bias, residual, wide)
    g = torch.Generator(device="cuda").manual_seed(M * 31 + N * 7 + K)
    x, w = rows(g, M, K, dtype), rows(g, N, K, dtype, K ** -0.5)
    kind = torch.float32 if wide else dtype
    b = normal(g, N, dtype=dtype) if bias else None
    ld = -(-N // 8) * 8
    r = normal(g, M, ld, dtype=kind)[:, :N] if residual else None
    whole = torch.full((M, ld), 7.0, dtype=kind, device="cuda")
    out = whole[:, :N]
    na.linear16(x, w, b, r, act, out)
    torch.cuda.synchronize()
    check(out, x, w, b, r, act, f"{M} x {N} x {K} {act}")
    assert (whole[:, N:] == 7.0).all()
    return out


@pytest.mark.parametrize("M,N,K,wide", PARTS)
@pytest.mark.parametrize("aligned", [False, True])
def test_epilogues_behind_parts(cuda_device, M, N, K, wide, aligned):
    for i, act in enumerate(na.ACTIVATIONS):
        for dtype in TYPES:
            padded(M, N, K, dtype, act, i % 2 == 0, i != 2, wide, aligned)
            padded(M, N, K, dtype, act, True, False, wide, aligned)
    assert na.linear16_status() == na.OK


@pytest.mark.parametrize("aligned", [False, True])
@pytest.mark.parametrize("act", list(na.ACTIVATIONS))
def test_epilogues_of_fp32_outputs(cuda_device, act, aligned):
    for M, N, K in ((4, 200, 256), (50, 200, 1024), (60, 1000, 2048), (300, 20000, 64), (4096, 8192, 128), (30000, 100, 64),
                    (1000, 1024, 4096), (400, 1004, 4096)):
        for bias, residual in ((False, False), (True, False), (False, True), (True, True)):
            padded(M, N, K, torch.bfloat16, act, bias, residual, True, aligned)


@pytest.mark.parametrize("M,N,K,wide", PARTS)
def test_sums_of_one_sign(cuda_device, M, N, K, wide):
    """What the tensor cores cut has one sign here (bounds as in the test of the same name in test_gpu_linear16)."""
    g = torch.Generator(device="cuda").manual_seed(K)
    x, w = (torch.zeros(n, -(-K // 8) * 8, dtype=torch.float16, device="cuda")[:, :K] for n in (M, N))
    x.copy_(0.5 + torch.rand(M, K, generator=g, device="cuda"))
    w.copy_((0.5 + torch.rand(N, K, generator=g, device="cuda")) / K)
    some = torch.randint(0, M, (500,), generator=g, device="cuda")
    kind, together = (torch.float32, 1024) if wide else (torch.float16, 16384)
    rel = na.linear16(x, w, out_dtype=kind)[some].double() / (x[some].double() @ w.double().T) - 1
    few = min(rel.numel(), 10000)
    assert abs(float(rel.mean())) <= min(K, together) * 2.0 ** -27 + (2 + K / 1024) * U + 4 * half_step(kind) / (3 * few) ** 0.5
    assert float(rel.abs().max()) <= min(K, together) * 2.0 ** -27 + (40 + K / 1024) * U + half_step(kind)


@pytest.mark.parametrize("M,N,K,wide", PARTS)
def test_runs_are_identical(cuda_device, M, N, K, wide):
    a = case(M, N, K, torch.bfloat16, wide=wide)
    for _ in range(2):
        assert torch.equal(a, case(M, N, K, torch.bfloat16, wide=wide))
