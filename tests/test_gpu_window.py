"""nllb_attn_window on the GPU against attention in 64 bits over the keys that each token sees.  The tolerances are those
of test_gpu_rows.py, whose arithmetic this is; what no token of a call sees is NaN, or not there at all."""
import math

import pytest
import torch

import nllb_attn as na
from test_gpu_rows import LENS, MANY, TYPES, Paged, check, ctx, half_step, ints, reference  # noqa: F401 (ctx is a fixture)

pytestmark = pytest.mark.gpu


def visible(n, p, window, sinks):
    """[n tokens, n + p keys]"""
    j, t = torch.arange(n + p)[None, :], p + torch.arange(n)[:, None]
    return (j <= t) & ((j > t - window) | (j < sinks))


class Window(Paged):
    """A paged cache with what nobody sees taken out: NaN in its slots, no entries for pages that hold nothing else."""

    def __init__(self, lens, heads, kv_heads, dim, page, dtype, window, sinks, seed=0, hnd=False, extra_rows=0):
        super().__init__(lens, heads, kv_heads, dim, page, dtype, seed, hnd, extra_rows)
        self.window, self.sinks = window, sinks
        keep = [torch.full_like(self.k_pages, math.nan), torch.full_like(self.v_pages, math.inf)]
        table = self.table.tolist()
        for i, (n, p) in enumerate(lens):
            seen = visible(n, p, window, sinks).any(0) if n else torch.zeros(p, dtype=torch.bool)
            for e in range(-(-(n + p) // page)):
                at = torch.arange(e * page, min(n + p, (e + 1) * page))
                live = seen[at] & (at < p)
                pg = table[i][e]
                slots = (at % page)[live].cuda()
                for to, of in zip(keep, (self.k_pages, self.v_pages)):
                    to[pg, slots] = of[pg, slots]
                if not (seen[at] | (at >= p)).any():
                    table[i][e] = -1
        self.k_pages.copy_(keep[0])
        self.v_pages.copy_(keep[1])
        self.table = ints(table)

    def run(self, ctx, new=True, **kw):
        a = ctx.window_args(self.q, self.k_pages, self.v_pages, self.table, self.kv_len, self.out, self.window, self.sinks,
                            k_new=self.k_new if new else None, v_new=self.v_new if new else None, q_start=self.q_start,
                            q_len=self.q_len, max_q=max(n for n, _ in self.lens),
                            max_kv=max(max(n + p for n, p in self.lens), 1), **kw)
        ctx.window(a)
        return a

    def verify(self, what=""):
        for i, (n, p) in enumerate(self.lens):
            if n == 0:
                continue
            k, v = self.keys(i, self.k_pages, self.k_new), self.keys(i, self.v_pages, self.v_new)
            a = self.starts[i]
            ref, tol = reference(self.q[a:a + n], k, v, visible(n, p, self.window, self.sinks), self.scale)
            check(self.out[a:a + n], ref, tol, f"{what} sequence {i} ({n} after {p}, {self.window} and {self.sinks})")


SEEN = [(1, 0), (1, 1), (2, 3), (33, 0), (64, 4), (100, 100), (513, 16), (5000, 2)]


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("window,sinks", SEEN)
@pytest.mark.parametrize("lens", LENS, ids=[k.replace(" ", "-") for k in LENS])
def test_window_matches_64_bits(ctx, lens, window, sinks, dtype):  # noqa: F811
    heads, kv_heads, dim = [(4, 4, 64), (6, 2, 64), (8, 1, 128), (2, 2, 128)][(window + sinks) % 4]
    c = Window(LENS[lens], heads, kv_heads, dim, 16, dtype, window, sinks, seed=window, extra_rows=3)
    before = c.k_pages.clone(), c.v_pages.clone()
    c.run(ctx)
    ctx.sync()
    c.verify(lens)
    assert (c.out[sum(n for n, _ in c.lens):] == 7.0).all()  # rows behind the last sequence
    k, v = c.k_pages.clone(), c.v_pages.clone()
    c.k_pages, c.v_pages = before
    c.append()
    for x, y in ((c.k_pages, k), (c.v_pages, v)):  # the chunk's slots and no others (NaN elsewhere)
        assert ((x == y) | (torch.isnan(x) & torch.isnan(y))).all()


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(5, 1, 64), (15, 5, 128), (3, 3, 64), (16, 1, 64)])
@pytest.mark.parametrize("window,sinks", [(40, 3), (200, 0)])
def test_shared_heads(ctx, heads, kv_heads, dim, window, sinks, dtype):  # noqa: F811
    for lens in ([(1, 300), (1, 39), (1, 40), (1, 0)], [(3, 100), (2, 41), (1, 500)], [(100, 90), (17, 1000), (300, 0)]):
        c = Window(lens, heads, kv_heads, dim, 16, dtype, window, sinks, seed=heads)
        c.run(ctx)
        ctx.sync()
        c.verify()


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 16, 64), (16, 16, 128), (24, 12, 64)])
def test_many_chunks(ctx, heads, kv_heads, dim, dtype):  # noqa: F811
    """Enough of them that a CTA takes two query tiles, whose rows start their windows 255 tokens apart."""
    c = Window(MANY, heads, kv_heads, dim, 32, dtype, 130, 7, seed=heads + dim)
    c.run(ctx)
    ctx.sync()
    c.verify("many chunks")


@pytest.mark.parametrize("page", [1, 7, 48, 128])
@pytest.mark.parametrize("hnd", [False, True], ids=["nhd", "hnd"])
@pytest.mark.parametrize("lens", ["tokens", "chunks"])
def test_page_sizes_and_layouts(ctx, page, hnd, lens):  # noqa: F811
    for dtype in (torch.float32, torch.bfloat16):
        c = Window(LENS[lens], 4, 2, 64, page, dtype, 60, 5, seed=page, hnd=hnd)
        c.run(ctx)
        ctx.sync()
        c.verify(f"pages of {page}")


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens", ["tokens", "short chunks", "chunks"])
def test_a_window_that_hides_nothing(ctx, lens, dtype):  # noqa: F811
    """As nllb_attn_paged, bit for bit, where max_kv says so; else within tolerances."""
    c = Paged(LENS[lens], 4, 2, 64, 16, dtype, seed=3)
    c.run(ctx)
    ctx.sync()
    first = c.out.clone()
    longest = max(n + p for n, p in c.lens)
    for window, sinks, equal in ((longest, 0, True), (2 ** 31 - 1, 2 ** 31 - 1, True), (1, longest, False), (longest - 1, 1, False)):
        c.out.fill_(7.0)
        ctx.window(ctx.window_args(c.q, c.k_pages, c.v_pages, c.table, c.kv_len, c.out, window, sinks, k_new=c.k_new,
                                   v_new=c.v_new, q_start=c.q_start, q_len=c.q_len, max_q=max(n for n, _ in c.lens),
                                   max_kv=longest))
        ctx.sync()
        c.verify(f"{window} {sinks}")
        assert not equal or torch.equal(first, c.out)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("chunk", [1, 5, 150])
def test_a_ring_of_pages(ctx, dtype, chunk):  # noqa: F811
    """A running translation whose pages go round: the pages behind the window take the new tokens."""
    window, sinks, page, H, D, total = 90, 3, 16, 2, 64, 700
    g = torch.Generator().manual_seed(chunk)
    q, k, v = (torch.randn(total, H, D, generator=g).to(dtype).cuda() for _ in range(3))
    ring = -(-(window + chunk + page) // page)
    n_entries = -(-total // page)
    table = ints([[0] + [1 + e % ring for e in range(n_entries - 1)]])  # the first page stays
    kp, vp = (torch.full((ring + 1, page, H, D), math.nan, dtype=dtype, device="cuda") for _ in range(2))
    out = torch.empty_like(q)
    for a in range(0, total, chunk):
        b = min(total, a + chunk)
        ctx.window(ctx.window_args(q[a:b], kp, vp, table, ints([b]), out[a:b], window, sinks, k_new=k[a:b], v_new=v[a:b]))
    ctx.sync()
    ref, tol = reference(q, k, v, visible(total, 0, window, sinks), D ** -0.5)
    check(out, ref, tol, f"ring, chunks of {chunk}")


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,dim", [(1, 64), (40, 64), (40, 128)])
def test_windows_of_very_many_keys(ctx, n, dim, dtype):  # noqa: F811
    c = Window([(n, 70000)], 2, 1, dim, 64, dtype, 45000, 100)
    c.run(ctx)
    ctx.sync()
    c.verify("very many")


def test_far_offsets(ctx):  # noqa: F811
    """Pages more than 2^31 elements into the cache, and positions far beyond what the cache holds."""
    page, pool = 16, 2 ** 31 // (16 * 64) + 64
    k = torch.full((pool, page, 1, 64), math.nan, dtype=torch.bfloat16, device="cuda")
    v = torch.full_like(k, math.nan)
    for n in (1, 130):
        past = 900000
        window, sinks = 100, 4
        c = Paged([(n, 100 + sinks)], 1, 1, 64, page, torch.bfloat16)  # the rows that are seen
        table = torch.full((1, -(-(past + n) // page)), -5, dtype=torch.int32)
        first = past - window + 1
        need = sorted({j // page for j in range(first, past + n)} | {0})
        for i, e in enumerate(need):
            table[0, e] = pool - 1 - 3 * i
        at = list(range(sinks)) + list(range(past - 100, past))
        rows = torch.randn(2, len(at), 1, 64).to(torch.bfloat16).cuda()
        for r, j in enumerate(at):
            if table[0, j // page] >= 0:
                k[int(table[0, j // page]), j % page], v[int(table[0, j // page]), j % page] = rows[0, r], rows[1, r]
        out = torch.empty_like(c.q)
        ctx.window(ctx.window_args(c.q, k, v, table.cuda(), ints([past + n]), out, window, sinks, k_new=c.k_new, v_new=c.v_new))
        ctx.sync()
        kk, vv = torch.cat([rows[0], c.k_new]), torch.cat([rows[1], c.v_new])
        j = torch.tensor(at + list(range(past, past + n)))
        t = past + torch.arange(n)[:, None]
        ref, tol = reference(c.q, kk, vv, (j <= t) & ((j > t - window) | (j < sinks)), c.scale)
        check(out, ref, tol, f"far, {n}")


@pytest.mark.parametrize("lens", [[(1, 500)], [(140, 500)]], ids=["token", "chunk"])
def test_bad_pages_are_reported(ctx, lens):  # noqa: F811
    c = Window(lens, 2, 2, 64, 16, torch.bfloat16, 100, 2)
    assert int(c.table[0, 10]) == -1  # (nobody's: never looked at)
    good = c.table.clone()
    c.table[0, 30] = c.pool
    c.run(ctx)
    with pytest.raises(na.NllbAttnError) as e:
        ctx.sync()
    assert e.value.status == na.EINVAL and "page" in str(e.value)
    c.table = good
    c.run(ctx)
    ctx.sync()
    c.verify("after the error")


def test_a_wait_that_runs_out(ctx):  # noqa: F811
    c = Window([(140, 500)], 2, 2, 64, 16, torch.bfloat16, 100, 2)
    ctx.test_expire_next_rows_wait()
    c.run(ctx)
    with pytest.raises(na.NllbAttnError) as e:
        ctx.sync()
    assert e.value.status == na.ETIMEOUT and (c.out == 7.0).all()
    c.run(ctx)
    ctx.sync()
    c.verify("after the timeout")


def test_graphs_side_by_side(ctx):  # noqa: F811
    cs = [Window(LENS["tokens"], 4, 2, 64, 16, torch.bfloat16, 50, 4, seed=1),
          Window(LENS["one chunk behind a cache"], 4, 2, 64, 16, torch.float16, 700, 4, seed=2)]
    streams = [torch.cuda.Stream() for _ in cs]
    graphs = []
    for c, st in zip(cs, streams):
        c.run(ctx)
        torch.cuda.synchronize()
        c.out.fill_(7.0)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            ctx.set_stream(torch.cuda.current_stream().cuda_stream)
            c.run(ctx)
        graphs.append(g)
    ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for c in cs:
        c.verify("replayed")
