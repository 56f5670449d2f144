"""Whose error a bounded wait of nllb_linear16 that gave up is, with several streams."""
import pytest
import torch

import nllb_attn as na

pytestmark = pytest.mark.gpu

# a cluster per tile, single CTAs, pairs
SIZES = [(60, 1000, 2048), (30000, 100, 64), (300, 20000, 64)]


def operands(M, N, K):
    x, w = torch.ones(M, K, dtype=torch.float16, device="cuda"), torch.ones(N, K, dtype=torch.float16, device="cuda")
    out = torch.full((M, N), 7.0, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    return x, w, out


@pytest.mark.parametrize("M,N,K", SIZES, ids=["cluster", "single", "pair"])
def test_a_stream_with_a_word_of_its_own(cuda_device, M, N, K):
    """A status taken on another stream first does not take the report away."""
    x, w, out = operands(M, N, K)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    word, other = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    na.linear16_test_expire_next_wait()
    na.linear16(x, w, out=out, stream=b.cuda_stream, error=word)
    good = na.linear16(x, w, stream=a.cuda_stream, error=other)
    b.synchronize()
    assert na.linear16_status(a.cuda_stream) == na.OK and na.linear16_status(b.cuda_stream) == na.OK
    assert int(word) != 0 and int(other) == 0 and (out == 7.0).all() and (good == K).all()
    word.zero_()
    torch.cuda.synchronize()
    na.linear16(x, w, out=out, stream=b.cuda_stream, error=word)
    b.synchronize()
    assert int(word) == 0 and (out == K).all()


def test_the_word_of_a_device(cuda_device):
    """Without one, a status on any of its streams reports it, once."""
    x, w, out = operands(*SIZES[0])
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    na.linear16_test_expire_next_wait()
    na.linear16(x, w, out=out, stream=b.cuda_stream)
    b.synchronize()
    assert na.linear16_status(a.cuda_stream) == na.ETIMEOUT
    assert na.linear16_status(b.cuda_stream) == na.OK and na.linear16_status(a.cuda_stream) == na.OK


def test_captured(cuda_device):
    """A graph's call reports into the word that it was captured with, on whatever stream it is replayed."""
    x, w, out = operands(*SIZES[0])
    word, graph, st = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    na.linear16(x, w)
    torch.cuda.synchronize()
    na.linear16_test_expire_next_wait()
    with torch.cuda.graph(graph):
        na.linear16(x, w, out=out, error=word)
    for stream in (st, torch.cuda.Stream()):
        word.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        assert int(word) != 0 and (out == 7.0).all()
    assert na.linear16_status() == na.OK
