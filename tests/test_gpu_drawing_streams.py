"""The drawing decoder's operators on a stream of the caller's: ordered after the inputs made there and before the reads
of the outputs, and captured from there."""
import pytest
import torch

import nllb_attn as na
from test_gpu_rows import CROSS, LENS, Cross, Paged
from test_gpu_sample import check, f32, i32, make

pytestmark = pytest.mark.gpu

LONG = 20_000_000  # cycles, about 10 ms: what the stream does before the inputs are there


def test_sample_follows_the_current_stream(cuda_device):
    lg, u = make(24, 20011, torch.float32, seed=11)
    k, p = i32([0, 50, 0] * 8), f32([0.9, 1.0, 1.0] * 8)
    late = torch.full_like(lg, -1.0)
    na.sample(late, u, top_k=k, top_p=p)  # (a kernel's first launch may wait for the device)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        torch.cuda._sleep(LONG)
        late.copy_(lg)
        tok, logp = na.sample(late, u, top_k=k, top_p=p)
        kept = tok.clone(), logp.clone()
    st.synchronize()
    check(lg, u, *kept, None, k, p, None, "on the current stream")


def test_sample_is_captured_from_the_current_stream(cuda_device):
    lg, u = make(5, 100003, torch.float32, seed=12)
    work = lg.clone()
    tok, logp = torch.empty(5, dtype=torch.int32, device="cuda"), torch.empty(5, device="cuda")
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        na.sample(work, u, out_tok=tok, out_logp=logp)
    for seed in (13, 14):
        lg, _ = make(5, 100003, torch.float32, seed=seed)
        work.copy_(lg)
        g.replay()
        torch.cuda.synchronize()
        check(lg, u, tok, logp, what="replayed")


def test_all_three_on_a_stream_of_the_callers(cuda_device):
    """Inputs made late on a side stream, the three operators there, outputs read there."""
    st = torch.cuda.Stream()
    with na.Context(0, n_layers=0, max_sentences=0) as ctx:
        ctx.set_stream(st.cuda_stream)
        for lens in ("tokens", "chunks"):
            c = Paged(LENS[lens], 4, 2, 64, 16, torch.bfloat16, seed=3)
            x = Cross(CROSS["rows"], 4, 4, 64, torch.float32, seed=4)
            lg, u = make(7, 8192, torch.bfloat16, seed=5)
            late = [torch.zeros_like(c.q), torch.zeros_like(x.q), torch.zeros_like(lg)]
            na.sample(late[2], u)  # (a kernel's first launch may wait for the device)
            torch.cuda.synchronize()
            cq, xq = c.q, x.q
            with torch.cuda.stream(st):
                torch.cuda._sleep(LONG)
                for to, of in zip(late, (cq, xq, lg)):
                    to.copy_(of)
                c.q, x.q = late[0], late[1]
                c.run(ctx)
                ctx.cross_rows(ctx.cross_rows_args(
                    x.q, x.k, x.v, x.out, i32([t for _, t in x.lens]), q_start=i32(x.qs[:-1]),
                    q_len=i32([n for n, _ in x.lens]), kv_start=i32(x.ks[:-1]), max_q=max(n for n, _ in x.lens),
                    max_kv=max(t for _, t in x.lens)))
                tok, logp = na.sample(late[2], u)
                c.out, x.out, tok, logp = c.out.clone(), x.out.clone(), tok.clone(), logp.clone()
            st.synchronize()
            ctx.sync()
            c.q, x.q = cq, xq
            c.verify("side stream")
            x.verify("side stream")
            check(lg, u, tok, logp, what="side stream")
