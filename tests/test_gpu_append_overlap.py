"""nllb_attn_append whose buffers lie beside one another in the same memory, and over one another (refused)."""
import pytest
import torch

import nllb_attn as na
from test_gpu_append import Append, frequencies
from test_gpu_rows import TYPES, ctx  # noqa: F401 (ctx is a fixture)

pytestmark = pytest.mark.gpu

LENS = [(3, 14), (0, 9), (17, 0), (1, 1), (33, 100)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("turned", ["in place", "beside"])
def test_columns_of_one_projection(ctx, dtype, turned):  # noqa: F811
    """q, k and v, and where q goes to, are columns of the same rows; the pages of both pools are pairs in one buffer."""
    h, g, d, page = 8, 2, 64, 16
    t = Append(LENS, h, g, d, page, dtype, seed=5)
    whole = torch.zeros(t.rows, (2 * h + 2 * g) * d, dtype=dtype, device="cuda")
    part = [whole[:, a * d:b * d].view(t.rows, b - a, d) for a, b in ((0, h), (h, h + g), (h + g, h + 2 * g), (h + 2 * g, 2 * h + 2 * g))]
    for to, x in zip(part, (t.q, t.k, t.v)):
        to.copy_(x)
    t.k, t.v = part[1], part[2]
    q_out = part[0] if turned == "in place" else part[3]
    pair = torch.stack([t.kp, t.vp], 1).contiguous()  # [pool][2][page][heads][dim]
    t.kp, t.vp = pair[:, 0], pair[:, 1]
    q = part[0].clone()
    freq = frequencies(d // 2)
    kw = dict(q_start=t.q_start, q_len=t.q_len, max_q=33)
    ctx.append(ctx.append_args(t.k, t.v, t.kp, t.vp, t.table, t.kv_len, q=part[0], q_out=q_out, inv_freq=freq, **kw))
    torch.cuda.synchronize()
    t.q, t.q_out = q, q_out
    t.verify(freq, "halves", turned)


@pytest.mark.parametrize("over", ["k_new", "v_new", "q", "pages of each other", "keys' pages over k_new", "values' pages over q_out",
                                  "a page's last value"])
def test_refused(ctx, over):  # noqa: F811
    h, g, d, page, rows, pool = 4, 4, 64, 16, 64, 8
    flat = torch.zeros(1 << 20, dtype=torch.bfloat16, device="cuda")

    def heads(at, n=h):
        return flat[at:at + rows * n * d].view(rows, n, d)

    def pages(at):
        return flat[at:at + pool * page * g * d].view(pool, page, g, d)

    size = 1 << 16
    q, k, v, out, kp, vp = heads(0), heads(size), heads(2 * size), heads(3 * size), pages(4 * size), pages(5 * size)
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    kv_len = torch.tensor([32, 32], dtype=torch.int32, device="cuda")

    def call():
        ctx.append(ctx.append_args(k, v, kp, vp, table, kv_len, q=q, q_out=out, max_q=32))

    call()
    if over == "k_new":
        out = heads(size + 256)
    elif over == "v_new":
        out = heads(2 * size - 8)
    elif over == "q":
        out = heads(256)
    elif over == "pages of each other":
        vp = pages(4 * size + 7 * page * g * d)
    elif over == "keys' pages over k_new":
        kp = pages(size + (rows - 1) * g * d)
    elif over == "values' pages over q_out":
        vp = pages(3 * size)
    else:
        q = heads(6 * size)
        out = heads(4 * size + pool * page * g * d - 8)
    with pytest.raises(na.NllbAttnError, match="overlap"):
        call()
    torch.cuda.synchronize()
    assert (flat == 0).all()
