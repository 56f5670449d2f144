"""A decoder that draws, step by step: chunk attention over a paged cache, cross-attention, projection, nllb_sample.
Every drawn token and its log-probability are held against the definition in 64 bits (test_gpu_sample.py) on the logits
that the GPU drew from, and the logits against the same decoder in 64 bits fed the drawn tokens."""
import numpy as np
import pytest
import torch

import nllb_attn as na
from test_gpu_rows import ctx, ints, reference  # noqa: F401 (ctx is a fixture)
from test_gpu_sample import check, f32, i32

pytestmark = pytest.mark.gpu

B, H, D, V, PAGE, STEPS = 5, 2, 64, 997, 16, 12
W = H * D
SRC, PREFIX = [9, 23, 1, 40, 17], [3, 1, 18, 11, 2]
SETTINGS = dict(t=[1.0, 0.7, 1.3, 0.0, 1.0], k=[0, 20, 5, 0, 1], p=[0.9, 1.0, 0.8, 1.0, 1.0], m=[0.0, 0.05, 0.0, 0.0, 0.0])


def test_every_drawn_token(ctx):  # noqa: F811
    g = torch.Generator().manual_seed(21)
    emb, head = torch.randn(V, W, generator=g) * 0.5, torch.randn(W, V, generator=g) * 0.3
    proj = [torch.randn(W, W, generator=g) * W ** -0.5 for _ in range(4)]
    ks, vs = (torch.randn(sum(SRC), H, D, generator=g) for _ in range(2))
    tokens = [torch.randint(0, V, (n,), generator=g).tolist() for n in PREFIX]
    u = (torch.randint(0, 4096, (STEPS, B), generator=g).float() + 0.5) / 4096
    table = torch.randperm(B * 3, generator=g).to(torch.int32).view(B, 3).cuda()
    kp, vp = (torch.full((B * 3, PAGE, H, D), float("nan"), device="cuda") for _ in range(2))
    cu, cks, cvs, chead = [x.cuda() for x in proj], ks.cuda(), vs.cuda(), head.cuda()
    kv_start = ints(np.cumsum([0] + SRC)[:-1].tolist())
    t, k, p, m = f32(SETTINGS["t"]), i32(SETTINGS["k"]), f32(SETTINGS["p"]), f32(SETTINGS["m"])

    def logits_in_64_bits(seq, b):
        x = emb.double()[seq]
        n, s0 = len(seq), sum(SRC[:b])
        q, kk, v = ((x @ w.double()).view(n, H, D) for w in proj[:3])
        a, _ = reference(q, kk, v, torch.tril(torch.ones(n, n, dtype=torch.bool)), D ** -0.5)
        y = x + a.view(n, W)
        c, _ = reference((y @ proj[3].double()).view(n, H, D), ks[s0:s0 + SRC[b]], vs[s0:s0 + SRC[b]],
                         torch.ones(n, SRC[b], dtype=torch.bool), D ** -0.5)
        return ((y + c.view(n, W)) @ head.double())[-1]

    new = [list(x) for x in tokens]
    drawn = set()
    for step in range(STEPS):
        lens = [len(x) for x in new]
        starts = np.cumsum([0] + lens)[:-1].tolist()
        x = emb[torch.tensor(sum(new, []))].cuda()
        q, kn, vn = ((x @ w).view(-1, H, D) for w in cu[:3])
        out, cout = torch.empty_like(q), torch.empty_like(q)
        held = ints([len(s) for s in tokens]), ints(starts), ints(lens), ints(SRC)
        ctx.paged(ctx.paged_args(q, kp, vp, table, held[0], out, k_new=kn, v_new=vn, q_start=held[1], q_len=held[2],
                                 max_q=max(lens)))
        y = x + out.view(-1, W)
        cq = (y @ cu[3]).view(-1, H, D)
        ctx.cross_rows(ctx.cross_rows_args(cq, cks, cvs, cout, held[3], q_start=held[1], q_len=held[2],
                                           kv_start=kv_start, max_q=max(lens), max_kv=max(SRC)))
        last = torch.tensor([s + n - 1 for s, n in zip(starts, lens)], device="cuda")
        logits = (y + cout.view(-1, W))[last] @ chead
        tok, logp = na.sample(logits, u[step].cuda(), temperature=t, top_k=k, top_p=p, min_p=m)
        ctx.sync()
        check(logits, u[step], tok, logp, t, k, p, m, f"step {step}")
        for b in range(B):
            # fp32 products of two layers of 128: relative 2^-24 * 128 of the terms' size, far below 1e-3
            assert (logits[b].double().cpu() - logits_in_64_bits(tokens[b], b)).abs().max() < 1e-3
        new = [[int(x)] for x in tok.cpu()]
        for b in range(B):
            tokens[b].append(new[b][0])
            drawn.add(new[b][0])
    assert len(drawn) > STEPS  # (not one token over and over)
    assert na.SAMPLE_TIMEOUT not in drawn and -1 not in drawn
