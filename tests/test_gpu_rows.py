"""nllb_attn_paged and nllb_attn_cross_rows on the GPU against attention in 64 bits.

Tolerances, derived from the arithmetic and set before the first run.  With u = 2^-24 (half a step of fp32) and, per
query row, A = max_j scale * sum_d |q_d k_jd|: a score is off by at most ds = (D + 8) u A (D roundings of the products'
sum, the scaling, the base change; the two-part fp16 form of fp32 drops terms below 2^-22 A = 4 u A), which changes a
normalised weight by a factor within 1 +- 2 ds; the exponential and its argument's rounding add 8 u; a running sum over
n keys in strips adds at most (n / 8 + 32) u, twice that where the tensor core truncates.  16-bit calls may round each
weight once: half a step of the type.  All of these scale with the largest |v|.  The output is rounded once: half a
step of the type, relative to the value."""
import ctypes
import math

import numpy as np
import pytest
import torch

import nllb_attn as na

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ctx(cuda_device):
    with na.Context(0, n_layers=0, max_sentences=0) as c:
        c.set_stream(torch.cuda.current_stream().cuda_stream or 1)
        yield c


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def reference(q, k, v, seen, scale):
    """q [n, H, D], k, v [t, G, D], seen [n, t] bool; (attention, tolerance) in 64 bits."""
    n, H, D = q.shape
    G = k.shape[1]
    out = torch.zeros(n, H, D, dtype=torch.float64)
    tol = torch.full((n, H, 1), 0.0, dtype=torch.float64)
    qd, kd, vd = q.double().cpu(), k.double().cpu(), v.double().cpu()
    seen = seen.cpu()
    some = seen.any(1)
    for h in range(H):
        g = h // (H // G)
        live = seen.any(0)
        kk = torch.where(live[:, None], kd[:, g], 0.0)
        vv = torch.where(live[:, None], vd[:, g], 0.0)
        s = (qd[:, h] @ kk.T) * scale
        a = (qd[:, h].abs() @ kk.abs().T * scale).masked_fill(~seen, 0).amax(1) if len(kk) else torch.zeros(n)
        s = s.masked_fill(~seen, -math.inf)
        if s.shape[1]:
            w = torch.exp(s - s.amax(1, keepdim=True).clamp(min=-1e300))
            w = torch.where(some[:, None], w / w.sum(1, keepdim=True), 0.0)
            out[:, h] = w @ vv
            vmax = vv.abs().max()
            ds = (D + 8) * U * a
            chain = 2 * (s.shape[1] / 8 + 32) * U
            rounding = 0.0 if q.dtype == torch.float32 else half_step(q.dtype)
            tol[:, h, 0] = vmax * (2 * ds + 8 * U + chain + rounding)
    return out, tol + half_step(q.dtype) * out.abs()


def normal(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).cuda()


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def check(out, ref, tol, what):
    err = (out.double().cpu() - ref).abs()
    assert torch.isfinite(out).all(), what
    bad = err > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {float((err / tol.clamp(min=1e-30)).max()):.2f} tolerances"


class Paged:
    """A paged cache of sequences with the given (new, past) lengths, and its inputs."""

    def __init__(self, lens, heads, kv_heads, dim, page, dtype, seed=0, hnd=False, extra_rows=0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.page, self.dtype = lens, page, dtype
        need = [-(-(n + p) // page) for n, p in lens]
        self.pool = sum(need) + 2
        perm = torch.randperm(self.pool, generator=g).tolist()
        width = max(max(need), 1)
        table, at = [], 0
        for n in need:
            table.append(perm[at:at + n] + [-7] * (width - n))
            at += n
        self.table = ints(table)
        rows = sum(n for n, _ in lens) + extra_rows
        self.q = normal(g, rows, heads, dim, dtype=dtype, scale=2.0)
        self.k_new, self.v_new = (normal(g, rows, kv_heads, dim, dtype=dtype) for _ in range(2))
        shape = (self.pool, kv_heads, page, dim) if hnd else (self.pool, page, kv_heads, dim)
        self.k_pages, self.v_pages = (normal(g, *shape, dtype=dtype) for _ in range(2))
        if hnd:
            self.k_pages, self.v_pages = self.k_pages.transpose(1, 2), self.v_pages.transpose(1, 2)
        self.q_len, self.kv_len = ints([n for n, _ in lens]), ints([n + p for n, p in lens])
        starts = np.cumsum([0] + [n for n, _ in lens])[:-1].tolist()
        self.starts, self.q_start = starts, ints(starts)
        self.out = torch.full_like(self.q, 7.0)
        self.scale = dim ** -0.5

    def keys(self, i, pages, new):
        n, p = self.lens[i]
        ids = self.table[i, :-(-(n + p) // self.page)].long()
        x = pages[ids].reshape(-1, *pages.shape[2:])[:n + p].clone()
        x[p:] = new[self.starts[i]:self.starts[i] + n]
        return x

    def verify(self, what=""):
        for i, (n, p) in enumerate(self.lens):
            if n == 0:
                continue
            k, v = self.keys(i, self.k_pages, self.k_new), self.keys(i, self.v_pages, self.v_new)
            seen = torch.arange(n + p)[None, :] <= (p + torch.arange(n))[:, None]
            a = self.starts[i]
            ref, tol = reference(self.q[a:a + n], k, v, seen, self.scale)
            check(self.out[a:a + n], ref, tol, f"{what} sequence {i} ({n} after {p})")

    def run(self, ctx, new=True, **kw):
        a = ctx.paged_args(self.q, self.k_pages, self.v_pages, self.table, self.kv_len, self.out,
                           k_new=self.k_new if new else None, v_new=self.v_new if new else None,
                           q_start=self.q_start, q_len=self.q_len, max_q=max(n for n, _ in self.lens),
                           max_kv=max(max(n + p for n, p in self.lens), 1), **kw)
        ctx.paged(a)
        return a

    def append(self):
        """What the call writes into the pages, in torch."""
        for i, (n, p) in enumerate(self.lens):
            for t in range(n):
                pg = int(self.table[i, (p + t) // self.page])
                self.k_pages[pg, (p + t) % self.page] = self.k_new[self.starts[i] + t]
                self.v_pages[pg, (p + t) % self.page] = self.v_new[self.starts[i] + t]


LENS = {
    "first token": [(1, 0)],
    "tokens": [(1, 0), (1, 1), (1, 62), (1, 63), (1, 64), (1, 700), (0, 5), (1, 129)],
    "one far token": [(1, 5000)],
    "short chunks": [(3, 0), (2, 17), (0, 0), (4, 300)],
    "chunks": [(130, 0), (1, 127), (128, 1), (77, 513), (0, 9), (257, 130)],
    "one chunk behind a cache": [(40, 2500)],
}


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (6, 2, 64), (8, 1, 128), (5, 1, 64), (2, 2, 128)])
@pytest.mark.parametrize("lens", LENS, ids=[k.replace(" ", "-") for k in LENS])
def test_paged_matches_64_bits(ctx, lens, heads, kv_heads, dim, dtype):
    c = Paged(LENS[lens], heads, kv_heads, dim, 16, dtype, seed=heads * 7 + dim, extra_rows=3)
    before = c.k_pages.clone(), c.v_pages.clone()
    c.run(ctx)
    ctx.sync()
    c.verify(lens)
    assert (c.out[sum(n for n, _ in c.lens):] == 7.0).all()  # rows behind the last sequence
    k, v = c.k_pages.clone(), c.v_pages.clone()
    c.k_pages, c.v_pages = before
    c.append()
    assert torch.equal(c.k_pages, k) and torch.equal(c.v_pages, v)  # the chunk's slots and no others


# enough (sequence, key head) pairs that a CTA takes two query tiles: tails of one row, of a whole and of half a tile
MANY = [(129, 0), (256, 300), (257, 3), (130, 1000), (384, 64), (300, 127), (1, 9), (0, 0), (200, 700), (385, 31)]


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 16, 64), (16, 16, 128), (24, 12, 64), (36, 12, 128)])
def test_paged_many_chunks(ctx, heads, kv_heads, dim, dtype):
    c = Paged(MANY, heads, kv_heads, dim, 32, dtype, seed=heads + dim)
    c.run(ctx)
    ctx.sync()
    c.verify("many chunks")


@pytest.mark.parametrize("page", [1, 7, 48, 128])
@pytest.mark.parametrize("hnd", [False, True], ids=["nhd", "hnd"])
@pytest.mark.parametrize("lens", ["tokens", "chunks"])
def test_paged_page_sizes_and_layouts(ctx, page, hnd, lens):
    for dtype in (torch.float32, torch.bfloat16):
        c = Paged(LENS[lens], 4, 2, 64, page, dtype, seed=page, hnd=hnd)
        c.run(ctx)
        ctx.sync()
        c.verify(f"pages of {page}")


@pytest.mark.parametrize("lens", ["tokens", "chunks"])
def test_paged_without_new_rows_equals_with(ctx, lens):
    c = Paged(LENS[lens], 4, 2, 64, 16, torch.bfloat16)
    c.run(ctx)
    ctx.sync()
    first = c.out.clone()
    k = c.k_pages.clone()
    c.out.fill_(7.0)
    c.run(ctx, new=False)  # the chunk is in the pages by now
    ctx.sync()
    assert torch.equal(first, c.out) and torch.equal(k, c.k_pages)


def test_paged_strided_rows(ctx):
    """q, k_new and v_new as columns of one projection's output, out inside a wider buffer."""
    c = Paged(LENS["chunks"], 4, 4, 64, 16, torch.float16)
    rows = c.q.shape[0]
    wide = torch.empty(rows, 3, 4, 64, dtype=torch.float16, device="cuda")
    wide[:, 0], wide[:, 1], wide[:, 2] = c.q, c.k_new, c.v_new
    c.q, c.k_new, c.v_new = wide[:, 0], wide[:, 1], wide[:, 2]
    buf = torch.full((rows, 6, 64), 7.0, dtype=torch.float16, device="cuda")
    c.out = buf[:, 1:5]
    c.run(ctx)
    ctx.sync()
    c.verify("strided")
    assert (buf[:, 0] == 7.0).all() and (buf[:, 5] == 7.0).all()


def test_paged_nan_behind_the_lengths(ctx):
    """Slots past a sequence's length, and pages of nobody, are never used."""
    for dtype in TYPES:
        for lens in ("tokens", "chunks"):
            c = Paged(LENS[lens], 2, 2, 64, 16, dtype)
            keep_k, keep_v = c.k_pages.clone(), c.v_pages.clone()
            c.k_pages.fill_(float("nan"))
            c.v_pages.fill_(float("inf"))
            for i, (n, p) in enumerate(c.lens):
                for j in range(p):
                    pg = int(c.table[i, j // 16])
                    c.k_pages[pg, j % 16], c.v_pages[pg, j % 16] = keep_k[pg, j % 16], keep_v[pg, j % 16]
            c.run(ctx)
            ctx.sync()
            c.verify("nan behind")


def test_paged_far_offsets(ctx):
    """Pages more than 2^31 elements into the cache."""
    page, pool = 16, 2 ** 31 // (16 * 64) + 64
    k = torch.empty(pool, page, 1, 64, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    c = Paged([(1, 40), (130, 300)], 1, 1, 64, page, torch.bfloat16)
    used = sorted({int(x) for x in c.table.flatten().tolist() if x >= 0})
    far = {pg: pool - 1 - i for i, pg in enumerate(used)}
    for pg, to in far.items():
        k[to], v[to] = c.k_pages[pg], c.v_pages[pg]
    c.table = ints([[far.get(x, x) for x in row] for row in c.table.tolist()])
    c.k_pages, c.v_pages = k, v
    c.run(ctx)
    ctx.sync()
    c.verify("far pages")


def test_paged_runs_are_identical(ctx):
    c = Paged(LENS["one chunk behind a cache"], 4, 2, 64, 16, torch.float32)
    c.run(ctx)
    ctx.sync()
    first = c.out.clone()
    for _ in range(3):
        c.run(ctx)
    ctx.sync()
    assert torch.equal(first, c.out)


@pytest.mark.parametrize("bad_page", [-1, 10 ** 6])
@pytest.mark.parametrize("lens", [[(1, 50)], [(140, 100)]], ids=["token", "chunk"])
def test_paged_bad_page_is_reported(ctx, bad_page, lens):
    c = Paged(lens, 2, 2, 64, 16, torch.bfloat16)
    good = c.table.clone()
    c.table[0, 1] = bad_page
    c.run(ctx)
    with pytest.raises(na.NllbAttnError) as e:
        ctx.sync()
    assert e.value.status == na.EINVAL and "page" in str(e.value)
    c.table = good
    c.run(ctx)
    ctx.sync()
    c.verify("after the error")


@pytest.mark.parametrize("what", ["q_len", "kv_len", "kv_short", "q_start", "q_start_negative"])
def test_paged_bad_length_is_reported_and_left_out(ctx, what):
    for n in (1, 140):
        c = Paged([(n, 30), (n, 50)], 2, 2, 64, 16, torch.float32)
        k = c.k_pages.clone()
        tensors = {"q_len": (c.q_len, n + 1), "kv_len": (c.kv_len, n + 51), "kv_short": (c.kv_len, n - 1),
                   "q_start": (c.q_start, c.q.shape[0] - n + 1), "q_start_negative": (c.q_start, -1)}
        t, value = tensors[what]
        t[0] = value
        c.run(ctx)
        with pytest.raises(na.NllbAttnError) as e:
            ctx.sync()
        assert e.value.status == na.EINVAL and "length" in str(e.value)
        assert (c.out[:n] == 7.0).all()
        c.lens = c.lens[1:]
        c.starts, c.table = c.starts[1:], c.table[1:]
        c.verify("the other sequence")
        del k


def test_paged_graph_replay(ctx):
    """Two graphs captured on one context, replayed on two streams at once."""
    cs = [Paged(LENS["tokens"], 4, 2, 64, 16, torch.bfloat16, seed=1),
          Paged(LENS["one chunk behind a cache"], 4, 2, 64, 16, torch.bfloat16, seed=2)]
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


class Cross:
    def __init__(self, lens, heads, kv_heads, dim, dtype, seed=0, hide=0.0):
        g = torch.Generator().manual_seed(seed)
        self.lens = lens
        rows, keys = sum(n for n, _ in lens), sum(t for _, t in lens)
        self.q = normal(g, rows + 2, heads, dim, dtype=dtype, scale=2.0)
        self.k, self.v = (normal(g, keys + 1, kv_heads, dim, dtype=dtype) for _ in range(2))
        self.qs = np.cumsum([0] + [n for n, _ in lens]).tolist()
        self.ks = np.cumsum([0] + [t for _, t in lens]).tolist()
        self.mask = (torch.rand(keys + 1, generator=g) >= hide).to(torch.uint8).cuda() if hide else None
        self.out = torch.full_like(self.q, 7.0)
        self.scale = dim ** -0.5

    def run(self, ctx):
        a = ctx.cross_rows_args(self.q, self.k, self.v, self.out, ints([t for _, t in self.lens]),
                                q_start=ints(self.qs[:-1]), q_len=ints([n for n, _ in self.lens]),
                                kv_start=ints(self.ks[:-1]), max_q=max(n for n, _ in self.lens),
                                max_kv=max(t for _, t in self.lens), key_mask=self.mask)
        ctx.cross_rows(a)
        torch.cuda.synchronize()

    def verify(self, what=""):
        for i, (n, t) in enumerate(self.lens):
            if n == 0:
                continue
            qs, ks = slice(self.qs[i], self.qs[i] + n), slice(self.ks[i], self.ks[i] + t)
            seen = torch.ones(n, t, dtype=torch.bool)
            if self.mask is not None:
                seen &= (self.mask[ks] != 0).cpu()[None, :]
            ref, tol = reference(self.q[qs], self.k[ks], self.v[ks], seen, self.scale)
            check(self.out[qs], ref, tol, f"{what} sequence {i} ({n} over {t})")
        assert (self.out[self.qs[-1]:] == 7.0).all()


CROSS = {
    "one row one key": [(1, 1)],
    "tokens": [(1, 18), (1, 512), (0, 3), (1, 0), (1, 129), (1, 64)],
    "rows": [(21, 74), (132, 130), (1, 5), (9, 0), (0, 4), (129, 128), (64, 257)],
    "long": [(300, 1500), (5, 2000)],
    "few rows over many keys": [(6, 6000)],
}


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (6, 2, 128), (12, 1, 64)])
@pytest.mark.parametrize("hide", [0.0, 0.3, 0.97])
@pytest.mark.parametrize("lens", CROSS, ids=[k.replace(" ", "-") for k in CROSS])
def test_cross_rows_matches_64_bits(ctx, lens, heads, kv_heads, dim, dtype, hide):
    c = Cross(CROSS[lens], heads, kv_heads, dim, dtype, seed=dim + heads, hide=hide)
    c.run(ctx)
    c.verify(lens)
    ctx.sync()


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 16, 64), (16, 16, 128), (24, 12, 64)])
@pytest.mark.parametrize("hide", [0.0, 0.3, 0.99])
def test_cross_rows_many_sequences(ctx, heads, kv_heads, dim, dtype, hide):
    c = Cross([(n, t) for n, t in MANY], heads, kv_heads, dim, dtype, seed=heads + dim, hide=hide)
    c.run(ctx)
    c.verify("many sequences")
    ctx.sync()


def test_cross_rows_hidden_keys_may_hold_anything(ctx):
    for dtype in TYPES:
        for lens in ("tokens", "rows"):
            c = Cross(CROSS[lens], 4, 2, 64, dtype, hide=0.4)
            hidden = c.mask == 0
            c.k[hidden] = float("nan")
            c.v[hidden] = float("inf")
            c.run(ctx)
            c.verify("hidden")


def test_cross_rows_nan_query_stays_in_its_row(ctx):
    for dtype in TYPES:
        for lens in ("tokens", "rows", "few rows over many keys"):
            c = Cross(CROSS[lens], 4, 2, 64, dtype)
            c.run(ctx)
            plain = c.out.clone()
            c.q[1, 1] = float("nan")
            c.run(ctx)
            assert torch.isnan(c.out[1, 1]).all()
            c.out[1, 1] = plain[1, 1]
            assert torch.equal(c.out, plain)


def test_cross_rows_nan_key_reaches_the_rows_that_see_it(ctx):
    for dtype in TYPES:
        for key in (0, 5, 6, 7, 70):  # whichever way its weight is taken
            c = Cross([(200, 74), (140, 90)], 4, 2, 64, dtype)
            c.run(ctx)
            plain = c.out.clone()
            c.k[key, 1] = float("nan")  # read by query heads 2 and 3 of the first sequence
            c.run(ctx)
            assert torch.isnan(c.out[:200, 2:]).all()
            c.out[:200, 2:] = plain[:200, 2:]
            assert torch.equal(c.out, plain)


def test_cross_rows_everything_hidden_gives_zeros(ctx):
    for dtype in TYPES:
        for n in (1, 200):
            c = Cross([(n, 150), (n, 40)], 2, 2, 64, dtype, hide=0.5)
            c.mask[:150] = 0
            c.run(ctx)
            assert (c.out[:n] == 0).all()
            c.verify()


def test_cross_rows_padded_batch_and_extreme_scores(ctx):
    """[batch][length] tensors without starts, and scores far apart (one key takes all the weight)."""
    for dtype in TYPES:
        for n in (1, 33):
            g = torch.Generator().manual_seed(3)
            B, L, H, D = 3, 70, 2, 64
            q = normal(g, B * n, H, D, dtype=dtype, scale=30.0)
            k, v = normal(g, B * L, H, D, dtype=dtype, scale=10.0), normal(g, B * L, H, D, dtype=dtype)
            out = torch.empty_like(q)
            lens = [70, 1, 44]
            ctx.cross_rows(ctx.cross_rows_args(q, k, v, out, ints(lens)))
            ctx.sync()
            for b in range(B):
                ref, tol = reference(q[b * n:(b + 1) * n], k[b * L:b * L + lens[b]], v[b * L:b * L + lens[b]],
                                     torch.ones(n, lens[b], dtype=torch.bool), D ** -0.5)
                check(out[b * n:(b + 1) * n], ref, tol, f"{dtype} batch {b}")


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,kv_heads", [([(40, 900)], 2), (MANY, 12)], ids=["cluster", "two-tiles"])
def test_bounded_wait_runs_out_and_context_recovers(ctx, lens, kv_heads, dtype):
    c = Paged(lens, kv_heads, kv_heads, 64, 16, dtype, seed=3)
    ctx.test_expire_next_rows_wait()
    c.run(ctx)
    with pytest.raises(na.NllbAttnError) as e:
        ctx.sync()
    assert e.value.status == na.ETIMEOUT
    assert (c.out == 7.0).all()
    c.run(ctx)
    ctx.sync()
    c.verify("after the timeout")


def test_cross_rows_on_another_stream(ctx):
    c = Cross(CROSS["rows"], 4, 4, 64, torch.float32)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    ctx.set_stream(st.cuda_stream)
    try:
        c.run(ctx)
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    c.verify()


def test_cross_rows_bad_length_is_reported(ctx):
    c = Cross([(4, 10), (4, 10)], 2, 2, 64, torch.float32)
    a = ctx.cross_rows_args(c.q, c.k, c.v, c.out, ints([10, 11]), q_start=ints([0, 4]), q_len=ints([4, 4]),
                            kv_start=ints([0, 11]), max_q=4, max_kv=11)
    ctx.cross_rows(a)
    with pytest.raises(na.NllbAttnError) as e:
        ctx.sync()
    assert e.value.status == na.EINVAL
    assert (c.out[4:8] == 7.0).all() and not (c.out[:4] == 7.0).all()


# ---- a decoder's steps, as a program uses the three operators --------------------------------------------------


def test_sampling_decoder_run(ctx):
    """A one-layer decoder over a paged cache: forced prefixes of different lengths in one chunk, then token by
    token -- self-attention, cross-attention, projection, drawing -- against the same steps in 64 bits fed the
    drawn tokens."""
    g = torch.Generator().manual_seed(5)
    B, H, D, V, page, steps = 3, 2, 64, 997, 16, 6
    W = H * D
    emb, head = torch.randn(V, W, generator=g) * 0.5, torch.randn(W, V, generator=g) * 0.3
    proj = [torch.randn(W, W, generator=g) * W ** -0.5 for _ in range(4)]
    src_len, prefix = [9, 23, 1], [3, 1, 18]
    ks, vs = (torch.randn(sum(src_len), H, D, generator=g) for _ in range(2))
    tokens = [torch.randint(0, V, (n,), generator=g).tolist() for n in prefix]
    u = torch.rand(steps, B, generator=g)
    table = torch.arange(B * 3, dtype=torch.int32).view(B, 3).flip(0).contiguous().cuda()
    kp, vp = (torch.full((B * 3, page, H, D), float("nan"), device="cuda") for _ in range(2))
    cu = [x.cuda() for x in proj]
    kv_start = ints(np.cumsum([0] + src_len)[:-1].tolist())

    def reference_logits(seq, b):
        x = emb.double()[seq]
        q, k, v = (x @ p.double() for p in proj[:3])
        n = len(seq)
        sees = torch.tril(torch.ones(n, n, dtype=torch.bool))
        a, _ = reference(q.view(n, H, D), k.view(n, H, D), v.view(n, H, D), sees, D ** -0.5)
        y = x + a.view(n, W)
        s0 = sum(src_len[:b])
        rows = slice(s0, s0 + src_len[b])
        c, _ = reference((y @ proj[3].double()).view(n, H, D), ks[rows], vs[rows],
                         torch.ones(n, src_len[b], dtype=torch.bool), D ** -0.5)
        return ((y + c.view(n, W)) @ head.double())[-1]

    new = [list(t) for t in tokens]
    for step in range(steps):
        lens = [len(t) for t in new]
        x = emb[torch.tensor(sum(new, []))].cuda()
        q, k, v = ((x @ p).view(-1, H, D) for p in cu[:3])
        starts = np.cumsum([0] + lens)[:-1].tolist()
        out = torch.empty_like(q)
        total = ints([len(t) for t in tokens])
        ctx.paged(ctx.paged_args(q, kp, vp, table, total, out, k_new=k, v_new=v, q_start=ints(starts),
                                 q_len=ints(lens), max_q=max(lens)))
        y = x + out.view(-1, W)
        cq, cout = (y @ cu[3]).view(-1, H, D), torch.empty_like(q)
        ctx.cross_rows(ctx.cross_rows_args(cq, ks.cuda(), vs.cuda(), cout, ints(src_len), q_start=ints(starts),
                                           q_len=ints(lens), kv_start=kv_start, max_q=max(lens),
                                           max_kv=max(src_len)))
        last = torch.tensor([s + n - 1 for s, n in zip(starts, lens)], device="cuda")
        logits = (y + cout.view(-1, W))[last] @ head.cuda()
        tok, logp = na.sample(logits, u[step].cuda(), top_k=ints([0, 20, 5]),
                              top_p=torch.tensor([0.9, 1.0, 1.0], device="cuda"))
        ctx.sync()
        for b in range(B):
            ref = reference_logits(tokens[b], b)
            # fp32 products of two layers of 128: relative 2^-24 * 128 of the terms' size, far below 1e-3
            assert (logits[b].double().cpu() - ref).abs().max() < 1e-3
        new = [[int(t)] for t in tok.cpu()]
        assert all(0 <= t[0] < V for t in new) and torch.isfinite(logp).all()
        for b in range(B):
            tokens[b].append(new[b][0])


def test_context_error_word_is_cleared(ctx):
    ctx.sync()
    assert ctypes.sizeof(na.PagedArgs) == 10 * 8 + 12 * 4 + 14 * 8
