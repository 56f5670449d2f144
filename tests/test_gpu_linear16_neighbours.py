"""nllb_linear16 whose operands and outputs lie beside one another in the same memory."""
import pytest
import torch

import nllb_attn as na
from test_gpu_linear16 import check, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K", [(1, 40, 64), (7, 500, 512), (60, 500, 2048), (300, 20000, 64), (5000, 104, 504), (1000, 1024, 4096)])
def test_columns_of_one_matrix(cuda_device, M, N, K):
    """x, residual and out are columns of the same rows."""
    g = torch.Generator(device="cuda").manual_seed(M)
    whole = normal(g, M, K + 2 * N + (-2 * N) % 8, dtype=torch.bfloat16)
    before = whole.clone()
    w = normal(g, N, K, dtype=torch.bfloat16, scale=K ** -0.5)
    x, residual, out = whole[:, :K], whole[:, K:K + N], whole[:, K + N:K + 2 * N]
    na.linear16(x, w, residual=residual, out=out)
    torch.cuda.synchronize()
    check(out, before[:, :K], w, None, before[:, K:K + N], "none")
    assert torch.equal(whole[:, :K + N], before[:, :K + N]) and torch.equal(whole[:, K + 2 * N:], before[:, K + 2 * N:])


def test_halves_of_one_buffer(cuda_device):
    """Rows of other lengths behind one another; a residual in its place whose single row has any stride."""
    g = torch.Generator(device="cuda").manual_seed(3)
    M, N, K = 50, 136, 1088
    flat = normal(g, M * K + M * N + N * K, dtype=torch.float16)
    x, out, w = flat[:M * K].view(M, K), flat[M * K:M * K + M * N].view(M, N), flat[M * K + M * N:].view(N, K)
    w *= K ** -0.5
    keep = out.clone()
    na.linear16(x, w, residual=out, out=out)
    torch.cuda.synchronize()
    check(out, x, w, None, keep, "none")
    one = torch.randn(1, N, device="cuda").half()
    keep = one.clone()
    na.linear16(x[:1], w, residual=one.as_strided((1, N), (N + 64, 1)), out=one)
    torch.cuda.synchronize()
    check(one, x[:1], w, None, keep, "none")


@pytest.mark.parametrize("residual", [False, True])
def test_refused_in_memory_that_is_there(cuda_device, residual):
    flat = torch.zeros(1 << 16, dtype=torch.float16, device="cuda")
    x, w = flat[:64 * 64].view(64, 64), torch.zeros(64, 64, dtype=torch.float16, device="cuda")
    out = flat[1 << 15:(1 << 15) + 64 * 64].view(64, 64)
    with pytest.raises(na.NllbAttnError, match="overlap"):
        if residual:
            na.linear16(x, w, residual=flat[(1 << 15):].as_strided((64, 64), (72, 1)), out=out)
        else:
            na.linear16(x, w, out=flat[32:32 + 64 * 64].view(64, 64))
    na.linear16(x, w, residual=out, out=out)
    torch.cuda.synchronize()
    assert (flat == 0).all()
