"""The hook that lets a wait of nllb_linear16 run out is for the next call and no later one."""
import ctypes

import pytest
import torch

import nllb_attn as na

pytestmark = pytest.mark.gpu


def run(M, N, K, out=None):
    x, w = torch.ones(M, K, dtype=torch.float16, device="cuda"), torch.ones(N, K, dtype=torch.float16, device="cuda")
    out = na.linear16(x, w, out=out)
    return na.linear16_status(), out


@pytest.mark.parametrize("M,N,K", [(17, 100, 1032), (33, 2080, 2048), (17, 64, 64), (17, 5000, 256), (64, 1152, 1088), (1000, 16, 200)])
def test_sizes_that_the_tensor_cores_take(cuda_device, M, N, K):
    na.linear16_test_expire_next_wait()
    status, _ = run(M, N, K)
    assert status == na.ETIMEOUT
    status, out = run(M, N, K)
    assert status == na.OK and (out == K).all()


def refused():
    a = na.Linear16Args(M=3, N=5, K=64, dtype=na.F32)
    assert na.load().nllb_linear16(ctypes.byref(a), None) == na.EINVAL


def no_arguments():
    assert na.load().nllb_linear16(None, None) == na.EINVAL


def no_word():
    assert na.load().nllb_linear16_reporting(ctypes.byref(na.Linear16Args()), None, None) == na.EINVAL


def no_rows():
    assert run(0, 100, 64)[0] == na.OK


def other_kernel():
    status, out = run(64, 1152, 1024)
    assert status == na.OK and (out == 1024).all()
    na.linear16_test_expire_next_wait()
    status, out = run(2, 100, 64)
    assert status == na.OK and (out == 64).all()


@pytest.mark.parametrize("call", [refused, no_arguments, no_word, no_rows, other_kernel])
def test_used_up(cuda_device, call):
    na.linear16_test_expire_next_wait()
    call()
    status, out = run(100, 1000, 2048)
    assert status == na.OK and (out == 2048).all()
