"""The hook that lets a wait of nllb_sample run out is for the next call and no later one."""
import ctypes

import pytest
import torch

import nllb_attn as na

pytestmark = pytest.mark.gpu


def refused():
    assert na.load().nllb_sample(ctypes.byref(na.SampleArgs(dtype=7)), None) == na.EINVAL


def no_arguments():
    assert na.load().nllb_sample(None, None) == na.EINVAL


def no_rows():
    na.sample(torch.empty(0, 100, device="cuda"), torch.empty(0, device="cuda"))


@pytest.mark.parametrize("call", [refused, no_arguments, no_rows])
def test_used_up(cuda_device, call):
    lg = torch.full((3, 256206), -100.0, device="cuda")
    lg[:, 77] = 100.0
    u = torch.full((3,), 0.5, device="cuda")
    na.sample_test_expire_next_wait()
    assert (na.sample(lg, u)[0] == na.SAMPLE_TIMEOUT).all()
    na.sample_test_expire_next_wait()
    call()
    assert (na.sample(lg, u)[0] == 77).all()
