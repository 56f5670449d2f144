"""Calls that name a stream and make their outputs: memory that the current stream's queued work still uses is not theirs."""
import pytest
import torch

import nllb_attn as na

pytestmark = pytest.mark.gpu


def linear16(stream):
    x, w = torch.ones(300, 64, dtype=torch.float16, device="cuda"), torch.ones(500, 64, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    return lambda: na.linear16(x, w, stream=stream), (300, 500), torch.float16, 64.0


def logprobs(stream):
    lg = torch.zeros(7, 1 << 16, device="cuda")
    target = torch.zeros(7, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    return lambda: na.logprobs(lg, target, entropy=False, stream=stream)[0], (7,), torch.float32, -16 * 0.6931471805599453


def sample(stream):
    lg, u = torch.full((9, 1000), -100.0, device="cuda"), torch.full((9,), 0.5, device="cuda")
    lg[:, 77] = 100.0
    out_logp = torch.empty(9, device="cuda")
    torch.cuda.synchronize()
    return lambda: na.sample(lg, u, out_logp=out_logp, stream=stream)[0], (9,), torch.int32, 77


@pytest.mark.parametrize("of", [linear16, logprobs, sample])
def test_a_block_that_the_current_stream_still_writes(cuda_device, of):
    side = torch.cuda.Stream()
    call, shape, kind, want = of(side.cuda_stream)
    first = call()  # (a kernel's first launch may wait for the device)
    torch.cuda.synchronize()
    for _ in range(3):
        held = [torch.empty(shape, dtype=kind, device="cuda") for _ in range(8)]
        torch.cuda._sleep(40_000_000)
        for h in held:
            h.fill_(3)
        places = {h.data_ptr() for h in held}
        del held, h
        out = call()
        assert out.data_ptr() not in places
        torch.cuda.synchronize()
        assert (out - want).abs().max() <= abs(want) * 2.0 ** -20
        assert out.shape == first.shape and out.dtype == kind
        torch.cuda.synchronize()


def test_captured_on_the_named_stream(cuda_device):
    x, w = torch.ones(300, 64, dtype=torch.float16, device="cuda"), torch.ones(500, 64, dtype=torch.float16, device="cuda")
    na.linear16(x, w)
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        out = na.linear16(x, w, stream=st.cuda_stream)
    graph.replay()
    torch.cuda.synchronize()
    assert (out == 64).all()
