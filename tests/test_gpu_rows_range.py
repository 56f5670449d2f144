"""fp32 attention of many rows (nllb_attn_paged, nllb_attn_cross_rows) over the range of fp32's sizes, on both sides of
the count of rows that chooses the kernel, against attention in 64 bits with the tolerances of test_gpu_rows.py (which
scale with the scores' terms and the largest |v|)."""
import pytest
import torch

from test_gpu_rows import Cross, Paged, check, ctx, reference  # noqa: F401 (ctx is a fixture)

pytestmark = pytest.mark.gpu

# sizes of q, k and v; q and k change against each other, so the scores stay of order 1
SIZES = [(1.0, 1.0, 1e-4), (1.0, 1.0, 1e5), (1.0, 1.0, 1e-6), (1e-4, 1e4, 1.0), (1e4, 1e-4, 1.0), (1e8, 1e-8, 1e-30),
         (1e-6, 1e6, 1e20), (7e4, 1e-5, 0.03), (0.02, 30.0, 0.02), (1e-20, 1e20, 2e4)]

LENS = [[(8, 60)], [(9, 60)], [(9, 0), (40, 100)], [(40, 900)], [(130, 300), (3, 500)]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "-".join(f"{x:g}" for x in s))
@pytest.mark.parametrize("lens", LENS, ids=["8-rows", "9-rows", "two", "cluster", "tiles"])
def test_sizes(ctx, lens, sizes):  # noqa: F811
    for dim in (64, 128):
        c = Paged(lens, 2, 2, dim, 16, torch.float32, seed=dim)
        x = Cross([(n, n + p) for n, p in lens], 2, 1, dim, torch.float32, seed=dim + 1, hide=0.2)
        for o in (c, x):
            o.q *= sizes[0]
        for t in (c.k_pages, c.k_new, x.k):
            t *= sizes[1]
        for t in (c.v_pages, c.v_new, x.v):
            t *= sizes[2]
        c.run(ctx)
        ctx.sync()
        c.verify(f"paged, heads of {dim}")
        x.run(ctx)
        ctx.sync()
        x.verify(f"cross, heads of {dim}")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,t", [(200, 700), (33, 1100), (300, 129)])
def test_rows_and_tiles_of_different_sizes(ctx, n, t, dim):  # noqa: F811
    """Query rows of 1e-6 to 1 among one another; the keys' and values' sizes change from one 128 to the next."""
    c = Cross([(n, t)], 2, 2, dim, torch.float32, seed=n)
    c.q[:n] *= (10.0 ** -(torch.arange(n) % 7).float()).cuda()[:, None, None]
    tile = torch.arange(t + 1) // 128
    k_size = torch.tensor([1.0, 1e-5, 0.01, 1e-9, 2.0, 0.3, 1e-3, 1.0, 1e-6])[tile]
    v_size = torch.tensor([1e-5, 1.0, 3e4, 1e-7, 1.0, 2e5, 1e-2, 1e-12, 5.0])[tile]
    c.k *= k_size.cuda()[:, None, None]
    c.v *= v_size.cuda()[:, None, None]
    c.run(ctx)
    ctx.sync()
    c.verify("mixed sizes")


def test_small_values_beside_an_unused_pool(ctx):  # noqa: F811
    """What nobody reads (other pages, slots behind the lengths) sets no size."""
    c = Paged([(40, 100)], 2, 2, 64, 16, torch.float32)
    keep_k, keep_v = c.k_pages.clone(), c.v_pages.clone()
    c.k_pages.fill_(1e30)
    c.v_pages.fill_(1e30)
    for j in range(100):
        pg = int(c.table[0, j // 16])
        c.k_pages[pg, j % 16], c.v_pages[pg, j % 16] = keep_k[pg, j % 16], keep_v[pg, j % 16] * 1e-5
    c.v_new *= 1e-5
    c.run(ctx)
    ctx.sync()
    c.verify("unused pages")


@pytest.mark.parametrize("dim", [64, 128])
def test_zeros(ctx, dim):  # noqa: F811
    """Rows and tiles of zeros among ordinary ones."""
    c = Cross([(150, 500), (20, 300)], 2, 2, dim, torch.float32)
    c.q[:40] = 0
    c.k[128:256] = 0
    c.v[256:384] = 0
    c.run(ctx)
    ctx.sync()
    c.verify("zeros")
    c.v.zero_()
    c.run(ctx)
    assert (c.out[:170] == 0).all()
    ref, tol = reference(c.q[:150], c.k[:500], c.v[:500], torch.ones(150, 500, dtype=torch.bool), c.scale)
    check(c.out[:150], ref, tol, "zero values")


@pytest.mark.parametrize("huge", [1e6, 1e18, 1e30])
@pytest.mark.parametrize("dim", [64, 128])
def test_huge_rows_leave_their_neighbours_alone(ctx, dim, huge):  # noqa: F811
    """Query rows of finite garbage (padding that nobody reads), and keys of a chunk's later tokens, change nothing in the
    rows beside and before them."""
    c = Paged([(150, 300), (33, 0)], 2, 2, dim, 16, torch.float32, seed=dim)
    c.run(ctx)
    ctx.sync()
    plain = c.out.clone()
    bad = [5, 16, 17, 100, 149]
    c.q[bad] = huge
    c.k_new[149] = huge  # (row 149's own token sees it)
    c.out.fill_(7.0)
    c.run(ctx)
    ctx.sync()
    others = [i for i in range(183) if i not in bad]
    ref, tol = [], []
    for i, (n, p) in enumerate(c.lens):
        k, v = c.keys(i, c.k_pages, c.k_new), c.keys(i, c.v_pages, c.v_new)
        seen = torch.arange(n + p)[None, :] <= (p + torch.arange(n))[:, None]
        a = c.starts[i]
        r, t = reference(c.q[a:a + n], k, v, seen, c.scale)
        ref.append(r), tol.append(t)
    ref, tol = torch.cat(ref), torch.cat(tol)
    check(c.out[others], ref[others], tol[others], "beside huge rows")
    assert torch.equal(c.out[others], plain[others])  # bit for bit: each of them is of ordinary size
