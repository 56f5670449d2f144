"""16-bit attention of several rows over many keys.

The tensor cores cut what they add to a sum: an addition of 16 keys' products loses less than one step of fp32, 2^-23 of
the sum, so n keys lose at most n/16 * 2^-23 = n 2^-27 of an output whose terms have one sign.  Up to 32768 keys that may
stand; beyond, blocks of keys are added in fp32 (128 keys lose less than 1e-6, rounded additions as many again).  The
values here are positive, so a loss has one sign and the mean of the relative errors shows it.  The roundings of the
weights average out over the keys.  The output's is at most half a step; the dimensions' values are of different sizes,
so the mean of at least 64 of them deviates by half a step / sqrt(3 * 64), of which four are allowed."""
import pytest
import torch

from test_gpu_rows import CROSS, MANY, Cross, Paged, ctx, half_step, ints  # noqa: F401 (ctx is a fixture)

pytestmark = pytest.mark.gpu


def errors(ctx, rows, heads, n, dim, dtype, shared=False):  # noqa: F811
    """Relative errors of some rows of some heads; `shared`: all heads read the keys of one."""
    g = torch.Generator(device="cuda").manual_seed(dim + rows)
    q = torch.randn(rows, heads, dim, device="cuda", generator=g).to(dtype)
    k = torch.randn(n, 1 if shared else heads, dim, device="cuda", generator=g).to(dtype).expand(n, heads, dim)
    own = 1 if shared else heads
    v = 0.5 + 0.5 * torch.rand(n, own, dim, device="cuda", generator=g)
    v = (v * (1 + torch.rand(1, own, dim, device="cuda", generator=g))).to(dtype).expand(n, heads, dim)
    out = torch.empty_like(q)
    ctx.cross_rows(ctx.cross_rows_args(q, k, v, out, torch.tensor([n], dtype=torch.int32, device="cuda")))
    ctx.sync()
    some = torch.arange(0, rows, max(1, rows // 50), device="cuda")
    errs = []
    for h in range(0, heads, max(1, heads // 5)):
        s = q[some, h].double() @ k[:, h].double().T * dim ** -0.5
        ref = torch.softmax(s, 1) @ v[:, h].double()
        errs.append((out[some, h].double() / ref - 1).flatten())
    return torch.cat(errs)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [20000, 32768, 32769, 200000])
@pytest.mark.parametrize("rows,heads", [(80, 1), (9500, 4)], ids=["cluster", "two-tiles"])
def test_sums_of_many_rows(ctx, rows, heads, n, dim, dtype):  # noqa: F811
    e = errors(ctx, rows, heads, n, dim, dtype)
    lost = n * 2.0 ** -27 if n <= 32768 else 1e-5
    assert float(e.abs().max()) <= lost + 2 * half_step(dtype) + 1e-5
    assert abs(float(e.mean())) <= lost + 4 * half_step(dtype) / (3 * 64) ** 0.5


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("rows,dim", [(4, 64), (16, 64), (8, 128)])
def test_sums_of_several_rows(ctx, rows, dim, dtype):  # noqa: F811
    """Enough heads (which share their keys) that nothing splits them further than among a CTA's warps."""
    e = errors(ctx, rows, 320, 300000, dim, dtype, shared=True)
    assert float(e.abs().max()) <= 1e-5 + 2 * half_step(dtype) + 1e-5
    assert abs(float(e.mean())) <= 1e-5 + 4 * half_step(dtype) / (3 * 64) ** 0.5


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_sums_of_several_rows_over_millions_of_keys(ctx, dtype):  # noqa: F811
    e = errors(ctx, 4, 1, 3_700_001, 64, dtype)
    assert float(e.abs().max()) <= 1e-5 + 2 * half_step(dtype) + 1e-5
    assert abs(float(e.mean())) <= 1e-5 + 4 * half_step(dtype) / (3 * 64) ** 0.5


BOUND = 40000  # max_kv only bounds the lengths: short sequences in a call that is built for long ones


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (6, 2, 128), (16, 16, 64), (24, 12, 128), (12, 1, 64)])
@pytest.mark.parametrize("hide", [0.0, 0.3, 0.99])
@pytest.mark.parametrize("lens", ["rows", "long", "many", "very long"])
def test_short_sequences_under_a_long_bound(ctx, lens, heads, kv_heads, dim, hide, dtype):  # noqa: F811
    sizes = {"many": MANY, "very long": [(140, 5000), (1, 2049), (20, 2048)]}.get(lens) or CROSS[lens]
    c = Cross(sizes, heads, kv_heads, dim, dtype, seed=dim + heads, hide=hide)
    ctx.cross_rows(ctx.cross_rows_args(c.q, c.k, c.v, c.out, ints([t for _, t in sizes]), q_start=ints(c.qs[:-1]),
                                       q_len=ints([n for n, _ in sizes]), kv_start=ints(c.ks[:-1]),
                                       max_q=max(n for n, _ in sizes), max_kv=BOUND, key_mask=c.mask))
    ctx.sync()
    c.verify(lens)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("heads,dim", [(4, 64), (16, 64), (16, 128)])
def test_rising_scores_under_a_long_bound(ctx, heads, dim, dtype):  # noqa: F811
    """Maxima that grow by far more than 2^8 from tile to tile, before and after the first sums have moved on."""
    sizes = [(150, 5000), (260, 3000), (40, 4500)]
    c = Cross(sizes, heads, heads, dim, dtype, seed=3)
    c.q = c.q.abs() * 0.25
    at = torch.cat([torch.arange(t) / 500.0 for _, t in sizes] + [torch.zeros(1)]).cuda()
    c.k = (c.k * 0.1 + at[:, None, None]).to(dtype)
    ctx.cross_rows(ctx.cross_rows_args(c.q, c.k, c.v, c.out, ints([t for _, t in sizes]), q_start=ints(c.qs[:-1]),
                                       q_len=ints([n for n, _ in sizes]), kv_start=ints(c.ks[:-1]), max_q=260,
                                       max_kv=BOUND))
    ctx.sync()
    c.verify("rising")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (16, 16, 64), (24, 12, 128)])
def test_paged_chunks_under_a_long_bound(ctx, heads, kv_heads, dim, dtype):  # noqa: F811
    c = Paged(MANY + [(100, 4000)], heads, kv_heads, dim, 32, dtype, seed=dim)
    wide = torch.full((c.table.shape[0], BOUND // 32), -9, dtype=torch.int32, device="cuda")
    wide[:, :c.table.shape[1]] = c.table
    c.table = wide
    ctx.paged(ctx.paged_args(c.q, c.k_pages, c.v_pages, wide, c.kv_len, c.out, k_new=c.k_new, v_new=c.v_new,
                             q_start=c.q_start, q_len=c.q_len, max_q=max(n for n, _ in c.lens)))
    ctx.sync()
    c.verify("long bound")
    c.out.fill_(7.0)
    ctx.test_expire_next_rows_wait()
    ctx.paged(ctx.paged_args(c.q, c.k_pages, c.v_pages, wide, c.kv_len, c.out, k_new=c.k_new, v_new=c.v_new,
                             q_start=c.q_start, q_len=c.q_len, max_q=max(n for n, _ in c.lens)))
    import nllb_attn as na
    with pytest.raises(na.NllbAttnError) as e:
        ctx.sync()
    assert e.value.status == na.ETIMEOUT and (c.out == 7.0).all()
