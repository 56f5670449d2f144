"""A decoder in 16 bits over a rolling paged cache, step by step: projections, rotation and append, attention through a
window, projections onto the residual stream, the vocabulary's logits, log-probabilities of the given next tokens.  Each
operator's output is held against its definition in 64 bits on the inputs that the GPU had, every step; the positions' pages
go round, and the tokens that named the languages stay."""
import math

import pytest
import torch

import nllb_attn as na
from test_gpu_append import frequencies, turned
from test_gpu_linear16 import check as check_linear
from test_gpu_logprobs import check as check_logprobs
from test_gpu_rows import check as check_rows
from test_gpu_rows import ctx, ints, reference  # noqa: F401 (ctx is a fixture)
from test_gpu_window import visible

pytestmark = pytest.mark.gpu

B, H, G, D, V, F = 3, 4, 2, 64, 5003, 512
W, KV = H * D, G * D
PAGE, WINDOW, SINKS, RING = 16, 40, 2, 7  # (a ring of seven pages behind the first one, which stays)
PREFIX, STEPS = [50, 1, 23], 90


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_scoring_of_long_translations(ctx, dtype):  # noqa: F811
    g = torch.Generator().manual_seed(5)

    def weight(n, k):
        return (torch.randn(n, k, generator=g) * k ** -0.5).to(dtype).cuda()

    emb = (torch.randn(V, W, generator=g) * 0.5).to(dtype).cuda()
    wq, wk, wv, wo, w1, w2, head = weight(W, W), weight(KV, W), weight(KV, W), weight(W, W), weight(F, W), weight(W, F), weight(V, W)
    b1 = (torch.randn(F, generator=g) * 0.1).to(dtype).cuda()
    given = [torch.randint(0, V, (n + STEPS + 1,), generator=g) for n in PREFIX]
    freq = frequencies(D // 2)
    most = max(PREFIX) + STEPS
    table = torch.stack([torch.tensor([0] + [1 + e % RING for e in range(-(-most // PAGE) - 1)]) + b * (RING + 1) for b in range(B)])
    table = table.to(torch.int32).cuda()
    kp, vp = (torch.full((B * (RING + 1), PAGE, G, D), math.nan, dtype=dtype, device="cuda") for _ in range(2))
    keys = [torch.zeros(most, G, D, dtype=torch.float64) for _ in range(B)]    # what was appended, turned
    values = [torch.zeros(most, G, D, dtype=torch.float64) for _ in range(B)]
    done = [0] * B
    total = torch.zeros(B, dtype=torch.float64)

    for step in range(STEPS):
        lens = [PREFIX[b] if step == 0 else 1 for b in range(B)]
        starts = [sum(lens[:b]) for b in range(B)]
        rows = sum(lens)
        tokens = torch.cat([given[b][done[b]:done[b] + lens[b]] for b in range(B)])
        x = emb[tokens.cuda()]
        q, k, v = na.linear16(x, wq), na.linear16(x, wk), na.linear16(x, wv)
        check_linear(q, x, wq, None, None, "none")
        q3, k3, v3 = q.view(rows, H, D), k.view(rows, G, D), v.view(rows, G, D)
        before = q3.clone()
        kv_len, q_len, q_start = ints([done[b] + lens[b] for b in range(B)]), ints(lens), ints(starts)
        kw = dict(q_start=q_start, q_len=q_len, max_q=max(lens))
        ctx.append(ctx.append_args(k3, v3, kp, vp, table, kv_len, q=q3, q_out=q3, inv_freq=freq, **kw))
        pos = torch.cat([torch.arange(done[b], done[b] + lens[b]) for b in range(B)])
        want, tol = turned(before, pos, freq, "halves")
        assert ((q3.double().cpu() - want).abs() <= tol).all(), f"step {step}: queries"
        want, tol = turned(k3, pos, freq, "halves")
        att = torch.empty_like(q3)
        ctx.window(ctx.window_args(q3, kp, vp, table, kv_len, att, WINDOW, SINKS, **kw))
        y = na.linear16(att.view(rows, W), wo, residual=x)
        check_linear(y, att.view(rows, W), wo, None, x, "none")
        z = na.linear16(y, w1, b1, act="gelu")
        check_linear(z, y, w1, b1, None, "gelu")
        y2 = na.linear16(z, w2, residual=y)
        check_linear(y2, z, w2, None, y, "none")
        last = torch.tensor([starts[b] + lens[b] - 1 for b in range(B)], device="cuda")
        hidden = y2[last]
        logits = na.linear16(hidden, head, out_dtype=torch.float32)
        check_linear(logits, hidden, head, None, None, "none")
        nxt = torch.stack([given[b][done[b] + lens[b]] for b in range(B)]).to(torch.int32).cuda()
        out = na.logprobs(logits, nxt, top_n=5)
        check_logprobs(logits, nxt, out, 5, f"step {step}")
        total += out[0].double().cpu()
        ctx.sync()
        assert na.linear16_status() == na.OK
        for b in range(B):
            a, n, p = starts[b], lens[b], done[b]
            stored = torch.stack([kp[int(table[b, j // PAGE]), j % PAGE] for j in range(p, p + n)])
            assert ((stored.double().cpu() - want[a:a + n]).abs() <= tol[a:a + n]).all(), f"step {step}: keys of {b}"
            keys[b][p:p + n], values[b][p:p + n] = stored.double().cpu(), v3[a:a + n].double().cpu()
            ref, at_most = reference(q3[a:a + n], keys[b][:p + n], values[b][:p + n], visible(n, p, WINDOW, SINKS), D ** -0.5)
            check_rows(att[a:a + n], ref, at_most, f"step {step}, sequence {b}")
            done[b] += n
    assert torch.isfinite(total).all() and (total < 0).all()
    assert min(done) > PAGE * (RING + 1) - WINDOW or max(done) > PAGE * (RING + 1)  # (the pages went round)
