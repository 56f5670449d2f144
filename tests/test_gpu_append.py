"""nllb_attn_append on the GPU against the rotation in 64 bits.

Tolerance, set before the first run.  With u = 2^-24: the part of a turn is rounded to fp32 (pi u at most in the angle), its
sine and cosine are off by 2 units in the last place (4 u), two products and a sum add 3 u: 11 u of |a| + |b|; positions up
to 2^30 put 2^-53 * 2^28 turns, below 4 u, on the angle.  So 16 u (|a| + |b|), and half a step of the type of the value:
relative to it in the type's normal range, and fp16's steps below 2^-14 are all 2^-24, so half a step is 2^-25 there
(bf16's and fp32's lie below 2^-133).  What is not turned is equal."""
import numpy as np
import pytest
import torch

import nllb_attn as na
from test_gpu_rows import TYPES, Paged, ctx, half_step, ints, normal  # noqa: F401 (ctx is a fixture)

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def turned(x, pos, freq, pairs):
    """x [rows, heads, dim] turned in 64 bits, and the tolerance of each value."""
    n = freq.numel()
    y, tol = x.double().cpu(), torch.zeros(x.shape, dtype=torch.float64)
    if n == 0:
        return y, tol
    ang = (pos.double().cpu()[:, None] * freq.double().cpu())[:, None]
    a, b = (slice(0, n), slice(n, 2 * n)) if pairs == "halves" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    u, v = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = u * ang.cos() - v * ang.sin(), v * ang.cos() + u * ang.sin()
    tol[..., a] = tol[..., b] = 16 * U * (u.abs() + v.abs())
    least = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    tol[..., :2 * n] += (half_step(x.dtype) * y[..., :2 * n].abs()).clamp(min=least)
    return y, tol


def frequencies(n, base=10000.0):
    return (base ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))).float().cuda()


class Append:
    """A paged cache of sequences with the given (new, past) lengths, and its inputs."""

    def __init__(self, lens, heads, kv_heads, dim, page, dtype, seed=0, hnd=False, extra_rows=0, q=True):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.page = lens, page
        held = [range(p // page, -(-(n + p) // page)) for n, p in lens]
        self.pool = sum(map(len, held)) + 2
        perm = torch.randperm(self.pool, generator=g).tolist()
        table = torch.full((len(lens), max(1, max(-(-(n + p) // page) for n, p in lens))), -7, dtype=torch.int32)
        for i, h in enumerate(held):
            for e in h:
                table[i, e] = perm.pop()
        self.table = table.cuda()
        self.rows = sum(n for n, _ in lens) + extra_rows
        self.q = normal(g, self.rows, heads, dim, dtype=dtype) if q else None
        self.q_out = torch.full_like(self.q, 7.0) if q else None
        self.k, self.v = (normal(g, self.rows, kv_heads, dim, dtype=dtype) for _ in range(2))
        shape = (self.pool, kv_heads, page, dim) if hnd else (self.pool, page, kv_heads, dim)
        pages = [normal(g, *shape, dtype=dtype) for _ in range(2)]
        self.kp, self.vp = (x.transpose(1, 2) if hnd else x for x in pages)
        self.starts = np.cumsum([0] + [n for n, _ in lens])[:-1].tolist()
        self.q_len, self.kv_len, self.q_start = ints([n for n, _ in lens]), ints([n + p for n, p in lens]), ints(self.starts)
        self.pos = torch.zeros(self.rows, dtype=torch.int32)
        for a, (n, p) in zip(self.starts, lens):
            self.pos[a:a + n] = torch.arange(p, p + n)
        self.before = self.kp.clone(), self.vp.clone()

    def run(self, ctx, freq=None, pairs="halves", **kw):
        kw = dict(dict(q_start=self.q_start, q_len=self.q_len, max_q=max(max(n for n, _ in self.lens), 1)), **kw)
        ctx.append(ctx.append_args(self.k, self.v, self.kp, self.vp, self.table, self.kv_len, q=self.q, q_out=self.q_out,
                                   inv_freq=freq, pairs=pairs, **kw))

    def verify(self, freq, pairs, what="", pos=None, left_out=()):
        freq = torch.zeros(0) if freq is None else freq
        pos = self.pos if pos is None else pos.cpu()
        want_k, want_v = (x.double().cpu() for x in self.before)
        tol_k = torch.zeros_like(want_k)
        yk, tk = turned(self.k, pos, freq, pairs)
        if self.q is not None:
            yq, tq = turned(self.q, pos, freq, pairs)
            want = torch.full_like(yq, 7.0)
            tol = torch.zeros_like(tq)
        for i, (a, (n, p)) in enumerate(zip(self.starts, self.lens)):
            if i in left_out:
                continue
            for t in range(n):
                pg, slot = int(self.table[i, (p + t) // self.page]), (p + t) % self.page
                want_k[pg, slot], tol_k[pg, slot] = yk[a + t], tk[a + t]
                want_v[pg, slot] = self.v[a + t].double().cpu()
            if self.q is not None:
                want[a:a + n], tol[a:a + n] = yq[a:a + n], tq[a:a + n]
        assert (self.vp.double().cpu() == want_v).all(), f"{what}: values"
        assert ((self.kp.double().cpu() - want_k).abs() <= tol_k).all(), f"{what}: keys"
        if self.q is not None:
            assert ((self.q_out.double().cpu() - want).abs() <= tol).all(), f"{what}: queries"


LENS = {
    "one": [(1, 0)],
    "tokens": [(1, 5), (1, 0), (1, 99), (1, 16), (1, 15), (1, 17), (1, 3000)],
    "chunks": [(3, 14), (0, 9), (17, 0), (1, 1), (33, 100), (0, 0), (5, 31)],
    "long": [(700, 3), (1, 5000), (301, 65)],
    "many": [(n % 5, 7 * n % 400) for n in range(1, 260)],
    "prompts": [(1500, 0), (1000, 77), (250, 1)],
    "one prompt among tokens": [(1, 40)] * 70 + [(2000, 3), (0, 7)] + [(1 + n % 3, n) for n in range(300)] + [(700, 0)],
    "a short prompt among tokens": [(1, 40)] * 7 + [(200, 3), (0, 7)] + [(1, n) for n in range(30)] + [(0, 0)],
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", list(LENS))
@pytest.mark.parametrize("heads,kv_heads,dim,page,rot,pairs", [
    (2, 2, 64, 16, 64, "halves"), (8, 2, 128, 16, 128, "halves"), (4, 4, 64, 7, 64, "neighbours"),
    (12, 1, 128, 64, 64, "neighbours"), (15, 5, 64, 1, 32, "halves"), (6, 3, 128, 48, 48, "halves"),
    (4, 2, 64, 16, 16, "neighbours"), (4, 2, 128, 16, 0, "halves")])
def test_append(ctx, dtype, lens, heads, kv_heads, dim, page, rot, pairs):  # noqa: F811
    c = Append(LENS[lens], heads, kv_heads, dim, page, dtype, seed=len(lens) + dim, extra_rows=3)
    freq = frequencies(rot // 2) if rot else None
    c.run(ctx, freq, pairs)
    ctx.sync()
    c.verify(freq, pairs, f"{lens} {dtype}")


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_places(ctx, dtype):  # noqa: F811
    """Heads before slots in a page, rows of a fused projection, queries turned in their place."""
    lens, H, G, D = LENS["chunks"], 6, 2, 64
    for pairs in ("halves", "neighbours"):
        c = Append(lens, H, G, D, 16, dtype, seed=5, hnd=True)
        fused = torch.cat([c.q.flatten(1), c.k.flatten(1), c.v.flatten(1)], 1)
        kept = c.q.clone()
        c.q = fused[:, :H * D].view(-1, H, D)
        c.k = fused[:, H * D:(H + G) * D].view(-1, G, D)
        c.v = fused[:, (H + G) * D:].view(-1, G, D)
        c.q_out = c.q
        freq = frequencies(D // 2)
        c.run(ctx, freq, pairs)
        ctx.sync()
        c.q, c.q_out = kept, fused[:, :H * D].view(-1, H, D)
        assert (fused[:, H * D:].double().cpu() == torch.cat([c.k.flatten(1), c.v.flatten(1)], 1).double().cpu()).all()
        c.verify(freq, pairs, f"fused {pairs}")


def test_without_queries(ctx):  # noqa: F811
    c = Append(LENS["chunks"], 4, 4, 64, 16, torch.bfloat16, q=False)
    freq = frequencies(32)
    c.run(ctx, freq)
    ctx.sync()
    c.verify(freq, "halves")


@pytest.mark.parametrize("dtype", TYPES)
def test_lengths_that_count_for_more_than_the_rows(ctx, dtype):  # noqa: F811
    """Without queries sequences may share rows, and a bad start leaves a long length standing: no block of another is lost."""
    freq = frequencies(32)
    for n in (60, 2400):  # (a token to a CTA, and four)
        lens = [(n, 3)] + [(1, 40)] * 40 + [(n, 20)] * 3
        c = Append(lens, 2, 2, 64, 16, dtype, seed=9, q=False)
        c.starts = [0] + list(range(n, n + 40)) + [0, 5, 2]
        c.rows = n + 40
        c.k, c.v = c.k[:c.rows], c.v[:c.rows]
        c.q_start = ints(c.starts)
        rot = torch.zeros(c.rows, dtype=torch.int32)  # (a shared row has one position for all)
        rot.copy_(torch.arange(c.rows) % 1000)
        c.run(ctx, freq, position=ints(rot.tolist()))
        ctx.sync()
        c.verify(freq, "halves", "shared rows", rot)
        c = Append([(n, 3)] * 12 + [(1, 40)] * 60 + [(n, 2)], 2, 2, 64, 16, dtype, seed=10)
        short = c.rows - 11 * n
        c.starts = [-1 - i for i in range(11)] + [0] + list(range(n, n + 60)) + [n + 60]
        c.q, c.q_out, c.k, c.v, c.rows = c.q[:short], c.q_out[:short], c.k[:short], c.v[:short], short
        c.pos = torch.zeros(short, dtype=torch.int32)
        for a, (m, past) in zip(c.starts, c.lens):
            if a >= 0:
                c.pos[a:a + m] = torch.arange(past, past + m)
        c.q_start = ints(c.starts)
        c.run(ctx, freq)
        with pytest.raises(na.NllbAttnError):
            ctx.sync()
        c.verify(freq, "halves", "bad starts", left_out=range(11))


@pytest.mark.parametrize("dtype", TYPES)
def test_far_positions(ctx, dtype):  # noqa: F811
    """Positions where an angle in 32 bits would be far off, given ones among them."""
    lens = [(2, 131070), (3, 999990), (1, 5)]
    c = Append(lens, 2, 2, 64, 4096, dtype, seed=8)
    freq = frequencies(32, 500000.0)
    c.run(ctx, freq)
    ctx.sync()
    c.verify(freq, "halves", "far")
    c.kp.copy_(c.before[0])
    pos = ints([2 ** 30, 2 ** 30 - 1, 0, -7, 123456789, 1])
    c.run(ctx, freq, position=pos)
    ctx.sync()
    c.verify(freq, "halves", "given", pos)


def test_rows_without_starts(ctx):  # noqa: F811
    c = Append([(4, 10), (4, 0), (4, 33)], 4, 2, 64, 16, torch.float16)
    freq = frequencies(32)
    c.run(ctx, freq, q_start=None, q_len=None, max_q=4)
    ctx.sync()
    c.verify(freq, "halves")


def test_bad_lengths_and_pages_are_left_out(ctx):  # noqa: F811
    freq = frequencies(32)
    c = Append([(2, 20), (3, 5), (4, 40), (1, 1), (2, 2)], 2, 2, 64, 16, torch.float32, seed=2)
    c.q_len[0] = 100       # more than max_q
    c.kv_len[2] = 3        # fewer keys than tokens
    c.q_start[3] = c.rows  # behind the rows
    c.run(ctx, freq)
    with pytest.raises(na.NllbAttnError) as e:
        ctx.sync()
    assert e.value.status == na.EINVAL
    c.verify(freq, "halves", left_out=(0, 2, 3))
    # a bad page: its tokens are turned and not stored, the others are
    c = Append([(20, 10), (2, 2)], 2, 2, 64, 16, torch.float32, seed=3)
    good = int(c.table[0, 1])
    c.table[0, 1] = c.pool
    c.run(ctx, freq)
    with pytest.raises(na.NllbAttnError):
        ctx.sync()
    c.table[0, 1] = good
    c.kp[good], c.vp[good] = c.kp[good].clone(), c.vp[good].clone()
    assert (c.kp[good] == c.before[0][good]).all() and (c.vp[good] == c.before[1][good]).all()
    c.before = tuple(b.clone() for b in c.before)
    yk, _ = turned(c.k, c.pos, freq, "halves")
    c.kp[good, :14], c.vp[good, :14] = yk[6:20].to(c.kp.dtype).cuda(), c.v[6:20]
    c.verify(freq, "halves", "bad page")
    ctx.sync()  # (the error is gone)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_reads_what_was_appended(ctx, dtype):  # noqa: F811
    """append, then attention over the cache without new rows: as attention that writes the turned rows itself."""
    for lens in ([(1, 40), (1, 0)], [(60, 33), (90, 0)]):
        c = Paged(lens, 4, 2, 64, 16, dtype, seed=6)
        freq = frequencies(32)
        pos = torch.cat([torch.arange(p, p + n) for n, p in lens])
        q, k = c.q.clone(), c.k_new.clone()
        ctx.append(ctx.append_args(c.k_new, c.v_new, c.k_pages, c.v_pages, c.table, c.kv_len, q=c.q, q_out=c.q,
                                   inv_freq=freq, q_start=c.q_start, q_len=c.q_len, max_q=max(n for n, _ in lens)))
        c.run(ctx, new=False)
        ctx.sync()
        for got, was in ((c.q, q), (c.keys(0, c.k_pages, c.k_new)[lens[0][1]:], None)):
            if was is not None:
                want, tol = turned(was, pos, freq, "halves")
                assert ((got.double().cpu() - want).abs() <= tol).all()
        # the attention over what lies in the cache now
        want, tol = turned(k, pos, freq, "halves")
        for i, (n, p) in enumerate(lens):
            ids = c.table[i, :-(-(n + p) // 16)].long()
            stored = c.k_pages[ids].reshape(-1, 2, 64)[p:n + p]
            a = c.starts[i]
            assert ((stored.double().cpu() - want[a:a + n]).abs() <= tol[a:a + n]).all()
            c.k_new[a:a + n] = stored
        c.verify("appended")


def test_on_a_stream_captured_and_replayed(cuda_device):
    st = torch.cuda.Stream()
    freq = frequencies(64)
    with na.Context(0, n_layers=0, max_sentences=0) as ctx:  # noqa: F811
        ctx.set_stream(st.cuda_stream)
        c = Append(LENS["long"], 8, 2, 128, 16, torch.bfloat16, seed=4)
        late, q = torch.zeros_like(c.q), c.q
        c.q = late
        c.run(ctx, freq)  # (a kernel's first launch may wait for the device)
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            torch.cuda._sleep(20_000_000)
            late.copy_(q)
            c.run(ctx, freq)
            c.q_out = c.q_out.clone()
        st.synchronize()
        c.verify(freq, "halves", "stream")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            ctx.set_stream(torch.cuda.current_stream().cuda_stream)
            c.run(ctx, freq)
        late.copy_(q.flip(0))
        c.k.copy_(c.k.flip(0))
        c.q_out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        c.verify(freq, "halves", "replayed")
