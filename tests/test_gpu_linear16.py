"""nllb_linear16 on the GPU against the product in 64 bits.

Tolerance, derived from the arithmetic and set before the first run.  With u = 2^-24 and A = sum |x w| + |bias|: products
of 16-bit values are exact in fp32, the tensor cores cut off less than a step of fp32 with every 16 of the summands that they
add, at most 1024 for fp32 outputs and 16384 for others (k 2^-27 A); warps, splits, those sums' sum and the bias add at most
40 + K / 1024 roundings (u A each).  The activations have slopes up to 1.2 and are off by 16 u of
their argument's size, the residual's sum is rounded once (u), and the result to its type: half a step, relative to it in
the normal range, at least 2^-25 in fp16."""
import math

import pytest
import torch

import nllb_attn as na
from test_gpu_rows import half_step

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float16, torch.bfloat16]


def activated(y, act):
    if act == "relu":
        return y.clamp(min=0)
    if act == "gelu":
        return y * torch.special.ndtr(y)
    if act == "gelu_tanh":
        return y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
    return y * torch.sigmoid(y) if act == "silu" else y


def check(out, x, w, bias, residual, act, what=""):
    K = x.shape[1]
    y, a = x.double() @ w.double().T, x.double().abs() @ w.double().abs().T
    if bias is not None:
        y, a = y + bias.double(), a + bias.double().abs()
    z = activated(y, act)
    together = min(K, 1024 if out.dtype == torch.float32 else 16384)
    tol = 1.2 * (together * 2.0 ** -27 + (40 + K / 1024) * U) * a + 16 * U * y.abs()
    if residual is not None:
        z = z + residual.double()
        tol += U * z.abs()
    least = 2.0 ** -25 if out.dtype == torch.float16 else 0.0
    tol += (half_step(out.dtype) * z.abs()).clamp(min=least)
    err = (out.double() - z).abs()
    assert torch.isfinite(out).all(), what
    bad = err > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {float((err / tol.clamp(min=1e-30)).max()):.2f} tolerances"


def normal(gen, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def rows(gen, n, k, dtype, scale=1.0):
    """[n][k] in rows of a multiple of 8, NaN behind them."""
    x = torch.full((n, -(-k // 8) * 8 + 8), math.nan, dtype=dtype, device="cuda")
    x[:, :k] = normal(gen, n, k, dtype=dtype, scale=scale)
    return x[:, :k]


def case(M, N, K, dtype, act="none", bias=True, residual=True, wide=False, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + M * 31 + N * 7 + K)
    x, w = rows(g, M, K, dtype), rows(g, N, K, dtype, K ** -0.5)
    kind = torch.float32 if wide else dtype
    b = normal(g, N, dtype=dtype) if bias else None
    r = normal(g, M, N, dtype=kind) if residual else None
    whole = torch.full((M, N + 3), 7.0, dtype=kind, device="cuda")  # (rows that start anywhere)
    out = whole[:, 1:N + 1]
    na.linear16(x, w, b, r, act, out)
    torch.cuda.synchronize()
    check(out, x, w, b, r, act, f"{M} x {N} x {K} {act}")
    assert (whole[:, 0] == 7.0).all() and (whole[:, N + 1:] == 7.0).all()
    return out


SIZES = [
    (1, 1, 1), (1, 16, 8), (2, 17, 7), (8, 100, 33), (9, 15, 100), (16, 1000, 1000), (1, 4096, 1024), (5, 1024, 4096),
    (13, 300, 8192), (3, 5003, 65), (40, 100, 1), (200, 33, 40), (70000, 5, 8),
    (17, 1, 64), (17, 128, 64), (31, 129, 100), (32, 127, 1000), (33, 1024, 4096), (64, 5003, 1024), (65, 256, 72), (100, 1000, 2048),
    (128, 128, 128), (129, 640, 513), (200, 300, 8192), (256, 20000, 96), (257, 1023, 1024), (1000, 1024, 512), (3000, 4099, 200),
    (10000, 1024, 64), (4097, 4096, 128), (300, 40001, 64), (1, 40000, 700), (16, 9001, 1000), (27, 1000, 1000), (32, 128, 8192),
    (20, 16, 72), (12, 2048, 4104), (3, 100, 70000), (30, 60, 33000), (100, 200, 40000), (300, 20000, 1100), (2100, 4000, 2500),
    (260, 300, 17000), (30000, 100, 64), (5000, 100, 500), (20000, 300, 600), (400, 1024, 4096), (700, 500, 3000), (250, 1000, 9000),
    (1000, 1023, 4100), (21, 127, 300), (140, 260, 400), (1500, 50, 800),
]


@pytest.mark.parametrize("dtype", TYPES, ids=["f16", "bf16"])
@pytest.mark.parametrize("wide", [False, True], ids=["same", "wide"])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_sizes(cuda_device, M, N, K, wide, dtype):
    case(M, N, K, dtype, wide=wide)
    assert na.linear16_status() == na.OK


@pytest.mark.parametrize("dtype", TYPES, ids=["f16", "bf16"])
@pytest.mark.parametrize("act", list(na.ACTIVATIONS))
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True), (True, True)])
def test_epilogues(cuda_device, act, bias, residual, dtype):
    """On each of the forms: few rows, and blocks of them, a cluster per tile, single CTAs, pairs."""
    for M, N, K in ((4, 200, 256), (50, 200, 1024), (60, 1000, 2048), (300, 20000, 64), (4096, 8192, 128), (30000, 100, 64),
                    (1000, 1024, 4096), (400, 1004, 4096)):
        case(M, N, K, dtype, act, bias, residual)


@pytest.mark.parametrize("M,N", [(4, 300), (30, 60), (100, 500), (600, 9000), (4096, 4096)])
@pytest.mark.parametrize("K", [1024, 2000, 8192, 40000])
def test_sums_of_one_sign(cuda_device, M, N, K):
    """What the tensor cores cut has one sign here, and shows in the mean: at most 1024 2^-27 for fp32 outputs, 16384 2^-27 for
    16-bit ones, whose roundings average out over 10000 and more outputs (half a step / sqrt(3 * 10000), four of it); the
    additions in fp32 round to nearest, 2^-24 at most with every 1024 summands."""
    g = torch.Generator(device="cuda").manual_seed(K)
    x = (0.5 + torch.rand(M, K, generator=g, device="cuda")).to(torch.float16)
    w = ((0.5 + torch.rand(N, K, generator=g, device="cuda")) / K).to(torch.float16)
    some = slice(0, 500)
    ref = x[some].double() @ w.double().T
    for kind, together in ((torch.float32, 1024), (torch.float16, 16384)):
        out = na.linear16(x, w, out_dtype=kind)
        rel = out[some].double() / ref - 1
        few = min(rel.numel(), 10000)
        assert abs(float(rel.mean())) <= min(K, together) * 2.0 ** -27 + (2 + K / 1024) * U + 4 * half_step(kind) / (3 * few) ** 0.5
        assert float(rel.abs().max()) <= min(K, together) * 2.0 ** -27 + (40 + K / 1024) * U + half_step(kind)


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_small_values_of_activations(cuda_device, act):
    """Far below 0 the result keeps its relative accuracy: 2^-18 allows for an argument off by 16 u of 9, whose slope in
    the exponent is up to 9 (gelu)."""
    x = torch.zeros(20, 64, dtype=torch.float16, device="cuda")
    x[:, 0] = -torch.linspace(0.5, 9, 20).to(torch.float16)
    w = torch.zeros(40, 64, dtype=torch.float16, device="cuda")
    w[:, 0] = 1
    for rows_ in (5, 20):
        out = torch.empty(rows_, 40, device="cuda")
        na.linear16(x[:rows_], w, act=act, out=out)
        y = x[:rows_, :1].double()
        want = {"gelu": 0.5 * y * torch.special.erfc(-y / math.sqrt(2)), "silu": y / (1 + torch.exp(-y)),
                "gelu_tanh": y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))}[act]
        rel = (out.double() / want - 1).abs()[(want.abs() > 1e-36).expand(-1, 40)]
        # gelu_tanh's exponent reaches 2 * 0.8 * 42 = 66, off by 16 u of it
        assert float(rel.max()) < (2.0 ** -13 if act == "gelu_tanh" else 2.0 ** -18) and len(rel)


@pytest.mark.parametrize("dtype", TYPES, ids=["f16", "bf16"])
@pytest.mark.parametrize("M,N,K", [(6, 96, 128), (40, 256, 640), (70, 900, 2560), (600, 9000, 64), (4096, 8192, 64), (400, 1024, 4096),
                                   (5000, 100, 504)])
def test_residual_in_place_and_strided_operands(cuda_device, M, N, K, dtype):
    g = torch.Generator(device="cuda").manual_seed(M)
    wide = normal(g, M, 3 * K, dtype=dtype)  # columns of a fused projection's output
    x, w = wide[:, K:2 * K], normal(g, N, K, dtype=dtype, scale=K ** -0.5)
    out = normal(g, M, N, dtype=dtype)
    before = out.clone()
    assert na.linear16(x, w, residual=out, out=out) is out
    torch.cuda.synchronize()
    check(out, x, w, None, before, "none")


@pytest.mark.parametrize("M,N,K", [(7, 500, 5000), (60, 500, 5000), (1000, 1024, 4096), (20000, 300, 600), (500, 20000, 300), (4096, 4096, 640)])
def test_runs_are_identical(cuda_device, M, N, K):
    a = case(M, N, K, torch.bfloat16, wide=True)
    for _ in range(3):
        assert torch.equal(a, case(M, N, K, torch.bfloat16, wide=True))


def test_nothing_to_do(cuda_device):
    x, w = torch.empty(0, 64, dtype=torch.float16, device="cuda"), torch.ones(5, 64, dtype=torch.float16, device="cuda")
    assert na.linear16(x, w).shape == (0, 5)


def test_infinities_and_nan_stay_in_their_places(cuda_device):
    """A NaN or infinite row of x, or of w, reaches its row, or column, alone."""
    for M, N, K in ((8, 96, 128), (40, 256, 640), (70, 900, 2560), (600, 9000, 64), (4096, 8192, 64)):
        g = torch.Generator(device="cuda").manual_seed(M)
        x, w = rows(g, M, K, torch.bfloat16), rows(g, N, K, torch.bfloat16)
        x[M // 2, 3], w[N // 3, 5] = math.nan, math.inf
        out = na.linear16(x, w)
        good = torch.ones(M, N, dtype=torch.bool, device="cuda")
        good[M // 2], good[:, N // 3] = False, False
        assert torch.isfinite(out[good]).all() and not torch.isfinite(out[~good]).any()


def test_streams_side_by_side_and_captured(cuda_device):
    cases = [(7, 1000, 1024), (60, 1000, 2048), (600, 9000, 128), (4096, 8192, 64)]
    g = torch.Generator(device="cuda").manual_seed(1)
    held = []
    for M, N, K in cases:
        x, w = rows(g, M, K, torch.bfloat16), rows(g, N, K, torch.bfloat16, K ** -0.5)
        out = na.linear16(x, w, act="silu")  # (a kernel's first launch may wait for the device)
        late, st, graph = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda"), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=st):
            na.linear16(late, w, act="silu", out=out)
        held.append((x, w, out, late, st, graph))
    torch.cuda.synchronize()
    for x, w, out, late, st, graph in held:
        out.fill_(7.0)
        with torch.cuda.stream(st):
            torch.cuda._sleep(20_000_000)
            late.copy_(x)
            for _ in range(3):
                graph.replay()
    torch.cuda.synchronize()
    for x, w, out, late, st, graph in held:
        check(out, x, w, None, None, "silu", "replayed")
    st = torch.cuda.Stream()
    for x, w, out, late, _, _ in held:
        late.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            torch.cuda._sleep(20_000_000)
            late.copy_(x)
            got = na.linear16(late, w)
            kept = got.clone()
        st.synchronize()
        check(kept, x, w, None, None, "none", "on the current stream")
    assert na.linear16_status() == na.OK


@pytest.mark.parametrize("M,N,K", [(60, 1000, 2048), (30000, 100, 64), (300, 20000, 64), (4096, 8192, 128)],
                         ids=["cluster", "single", "pair", "pairs"])
def test_a_wait_that_runs_out(cuda_device, M, N, K):
    g = torch.Generator(device="cuda").manual_seed(2)
    x, w = rows(g, M, K, torch.float16), rows(g, N, K, torch.float16, K ** -0.5)
    out = torch.full((M, N), 7.0, dtype=torch.float16, device="cuda")
    na.linear16_test_expire_next_wait()
    na.linear16(x, w, out=out)
    assert na.linear16_status() == na.ETIMEOUT
    assert (out == 7.0).all()
    assert na.linear16_status() == na.OK  # read once
    na.linear16(x, w, out=out)
    assert na.linear16_status() == na.OK
    check(out, x, w, None, None, "none", "after the timeout")
