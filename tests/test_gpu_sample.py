"""nllb_sample on the GPU against the definition in 64 bits (numpy, one row at a time).

Tokens have to be equal.  The kernel's weights are off by at most 2^-45 of the largest each (and by 2^-50 relative),
so a running sum of 256206 of them is off by less than 1e-8 of the largest weight: `draw` reports how near the drawn
token's borders u lies, and the tests' fixed inputs keep every u further away than that (checked here, in the
reference).  Log-probabilities are rounded once to fp32 from fp64: 2^-24 relative, plus 1e-8."""
import numpy as np
import pytest
import torch

import nllb_attn as na

pytestmark = pytest.mark.gpu

LEAST = 2.0 ** -45


def draw(lg, u, t=1.0, k=0, p=1.0, m=0.0):
    """(token, log-probability, margin of u) of one row."""
    lg = np.where(np.isnan(lg), -np.inf, lg.astype(np.float64))
    best = lg.max()
    if best == -np.inf or not (0 <= t < np.inf):
        return -1, -np.inf, 1.0
    if t == 0:
        return int(np.argmax(lg)), 0.0, 1.0
    t, k, p, m, u = np.float64(np.float32(t)), int(k), float(np.float32(p)), float(np.float32(m)), float(np.float32(u))
    with np.errstate(invalid="ignore", over="ignore"):
        x = np.where(lg == best, 0.0, (lg - best) / max(t, 2.0 ** -100))
    w = np.exp(x)
    w[w < LEAST] = 0
    order = np.lexsort((np.arange(len(lg)), -lg))
    if 0 < k < len(lg):
        order = order[:k]
    margin = 1.0
    if p < 1:
        c = np.cumsum(w[order])
        n = int(np.searchsorted(c, max(p, 0.0) * c[-1], side="left")) + 1
        order = order[:max(1, n)]
    if m > 0:
        keep = w[order] >= min(m, 1.0)
        keep[0] = True
        order = order[keep]
    idx = np.sort(order)
    idx = idx[w[idx] > 0]
    c = np.cumsum(w[idx])
    u = min(max(u, 0.0), 1.0) if u == u else 0.0
    j = min(int(np.searchsorted(c, u * c[-1], side="right")), len(idx) - 1)
    lo, hi = (c[j - 1] if j else -1.0), (c[j] if j + 1 < len(idx) else np.inf)
    margin = min(u * c[-1] - lo, hi - u * c[-1])
    return int(idx[j]), float(x[idx[j]] - np.log(c[-1])), margin


def check(logits, u, tok, logp, t=None, k=None, p=None, m=None, what=""):
    lg = logits.float().cpu().numpy()
    tok, logp, u = tok.cpu().numpy(), logp.cpu().numpy(), u.cpu().numpy()
    for r in range(len(lg)):
        s = [d if x is None else x[r].item() for x, d in ((t, 1.0), (k, 0), (p, 1.0), (m, 0.0))]
        rt, rl, margin = draw(lg[r], u[r], *s)
        assert margin > 1e-8, f"{what} row {r}: choose another u"
        assert tok[r] == rt, f"{what} row {r} {s}: {tok[r]} instead of {rt} (margin {margin:.2e})"
        if np.isfinite(rl):
            assert abs(logp[r] - rl) <= 2.0 ** -24 * abs(rl) + 1e-8, f"{what} row {r}: {logp[r]} instead of {rl}"
        else:
            assert logp[r] == rl


def f32(v):
    return torch.tensor(v, dtype=torch.float32, device="cuda")


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def make(rows, vocab, dtype, seed, spread=2.5, ld=None):
    g = torch.Generator().manual_seed(seed)
    lg = torch.randn(rows, vocab, generator=g) * spread
    buf = torch.full((rows, ld or vocab), 1e4, dtype=dtype)
    buf[:, :vocab] = lg.to(dtype)
    # whole 2^-12ths and a half: off the borders of small cases by construction
    u = (torch.randint(0, 4096, (rows,), generator=g).float() + 0.5) / 4096
    return buf.cuda()[:, :vocab], u.cuda()


SETTINGS = [dict(), dict(k=1), dict(k=7), dict(k=300), dict(p=0.9), dict(p=0.3), dict(p=0.999), dict(m=0.05),
            dict(k=40, p=0.8), dict(k=5000, p=0.95, m=0.001), dict(t=0.0), dict(t=0.3, p=0.95), dict(t=4.0, k=50),
            dict(p=0.0), dict(m=1.0), dict(k=10 ** 6, p=2.0, m=-1.0), dict(t=2.0, p=0.5, m=0.9)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 33, 1000, 8192, 8193, 20011, 100003, 256206])
def test_settings_match_64_bits(cuda_device, vocab, dtype):
    rows = len(SETTINGS)
    lg, u = make(rows, vocab, dtype, seed=vocab % 1000 + 1, ld=vocab + (8 - vocab) % 8)
    col = lambda key, d: [s.get(key, d) for s in SETTINGS]  # noqa: E731
    t, k, p, m = f32(col("t", 1.0)), i32(col("k", 0)), f32(col("p", 1.0)), f32(col("m", 0.0))
    before = lg.clone()
    tok, logp = na.sample(lg, u, temperature=t, top_k=k, top_p=p, min_p=m)
    torch.cuda.synchronize()
    assert torch.equal(lg, before)
    check(lg, u, tok, logp, t, k, p, m, f"vocab {vocab}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [66000, 70003])
def test_many_rows(cuda_device, vocab, dtype):
    """More than 64 MB of rows (which are read in every pass), of every setting, some with NaN, infinities and ties."""
    rows = 30 * len(SETTINGS)
    assert rows * vocab * dtype.itemsize >= 2 ** 26
    lg, u = make(rows, vocab, dtype, seed=5, ld=vocab + (8 - vocab) % 8)
    lg[3, ::5] = float("nan")
    lg[20] = -float("inf")
    lg[21, 100], lg[21, 65000] = float("inf"), float("inf")
    lg[22:40] = lg[22:40].round()  # thousands of equal logits
    lg[40, 5:] = -float("inf")
    col = lambda key, d: [s.get(key, d) for s in SETTINGS] * 30  # noqa: E731
    t, k, p, m = f32(col("t", 1.0)), i32(col("k", 0)), f32(col("p", 1.0)), f32(col("m", 0.0))
    before = lg.clone()
    tok, logp = na.sample(lg, u, temperature=t, top_k=k, top_p=p, min_p=m)
    torch.cuda.synchronize()
    assert torch.equal(lg.nan_to_num(7.5), before.nan_to_num(7.5))
    some = list(range(42)) + list(range(42, rows, 5))  # (every setting: 5 and their number have no common factor)
    check(lg[some], u[some], tok[some], logp[some], t[some], k[some], p[some], m[some], f"vocab {vocab}")
    again = na.sample(lg, u, temperature=t, top_k=k, top_p=p, min_p=m)
    few = na.sample(lg[:40], u[:40].contiguous(), temperature=t[:40].contiguous(), top_k=k[:40].contiguous(),
                    top_p=p[:40].contiguous(), min_p=m[:40].contiguous())
    assert torch.equal(again[0], tok) and torch.equal(again[1], logp)
    assert torch.equal(few[0], tok[:40]) and torch.equal(few[1], logp[:40])


@pytest.mark.parametrize("rows,dtype", [(1, torch.float32), (3, torch.bfloat16), (34, torch.float32)],
                         ids=["one", "few", "many"])
def test_largest_vocabulary(cuda_device, rows, dtype):
    V = 524288
    lg, u = make(rows, V, dtype, seed=rows)
    k = i32([(0, 50, 3000)[r % 3] for r in range(rows)])
    p = f32([(0.9, 1.0)[r % 2] for r in range(rows)])
    tok, logp = na.sample(lg, u, top_k=k, top_p=p)
    torch.cuda.synchronize()
    check(lg, u, tok, logp, None, k, p, None, "largest")
    flat = torch.zeros(rows, V, dtype=dtype, device="cuda")  # the largest sum of weights
    tok, logp = na.sample(flat, u)
    assert tok.tolist() == [int(x * V) for x in u.double().tolist()]
    assert (logp.double() + np.log(V)).abs().max() < 1e-6


def test_defaults_and_unaligned_rows(cuda_device):
    for dtype in (torch.float32, torch.bfloat16):
        lg, u = make(5, 20011, dtype, seed=3, ld=20013)  # rows at odd addresses
        tok, logp = na.sample(lg, u)
        torch.cuda.synchronize()
        check(lg, u, tok, logp)
        one = lg[2:3, 1:]
        tok, logp = na.sample(one, u[2:3])
        torch.cuda.synchronize()
        check(one, u[2:3], tok, logp)


def test_ties_go_to_the_lowest_index(cuda_device):
    """Equal logits: cuts keep the lowest indices, whatever the share of equal ones."""
    V = 40000
    rows = []
    for kind in range(4):
        lg = np.zeros(V, np.float32) if kind == 0 else np.full(V, -3.0, np.float32)
        if kind == 1:
            lg[100::7] = 2.0
        if kind == 2:
            lg[5], lg[30000] = 0.0, -0.0
        if kind == 3:
            lg[::2] = np.float32(1.5)
            lg[1::2] = np.nextafter(np.float32(1.5), np.float32(0))
        rows += [lg] * 4
    u = f32([0.1234, 0.7, 0.9997, 0.333] * 4)
    k = i32([1, 3, 250, 0] * 4)
    p = f32([1.0, 1.0, 0.77, 0.31] * 4)
    lg = torch.from_numpy(np.stack(rows)).cuda()
    tok, logp = na.sample(lg, u, top_k=k, top_p=p)
    torch.cuda.synchronize()
    check(lg, u, tok, logp, None, k, p, None, "ties")
    g = na.sample(lg, u, temperature=f32([0.0] * 16))[0]
    assert g.tolist() == [0] * 4 + [100] * 4 + [5] * 4 + [0] * 4


def test_infinities_nan_and_unusable_rows(cuda_device):
    V = 9001
    lg, _ = make(12, V, torch.float32, seed=9)
    lg[0] = -float("inf")
    lg[1] = float("nan")
    lg[2, 10:] = -float("inf")
    lg[3, ::3] = float("nan")
    lg[4, 17] = lg[4, 8000] = float("inf")
    lg[5] = -3.0e38
    lg[5, 4000] = 3.0e38
    u = f32([0.3, 0.3, 0.77, 0.41, 0.75, 0.5, 0.2, 0.2, 0.2, 0.6, 0.31, 0.43])
    t = f32([1, 1, 1, 1, 1, 1, -1.0, float("inf"), float("nan"), 1e-30, 1e30, 1e-39])
    p = f32([0.9, 0.9, 0.9, 0.9, 1.0, 0.9, 0.9, 0.9, 0.9, 0.9, 0.9, 0.9])
    tok, logp = na.sample(lg, u, temperature=t, top_p=p)
    torch.cuda.synchronize()
    assert tok[[0, 1, 6, 7, 8]].tolist() == [-1] * 5 and tok[4].item() == 8000
    # masks of the type's lowest value, and logits so large that their neighbours lie many temperatures away
    low = torch.full((4, V), torch.finfo(torch.float32).min, device="cuda")
    low[1, 70:] = -float("inf")
    low[2, 50], low[2, 60] = 2.0 ** 30, 2.0 ** 30 - 64
    low[3] = torch.linspace(1e10, 1e10 + 1e6, V)
    v = f32([0.50123, 0.50123, 0.999, 0.40123])
    for kw in (dict(), dict(top_p=f32([0.7] * 4)), dict(top_k=i32([30] * 4)), dict(temperature=f32([1, 1, 20, 900]))):
        check(low, v, *na.sample(low, v, **kw), *[kw.get(n) for n in ("temperature", "top_k", "top_p", "min_p")],
              what="far apart")
    check(lg, u, tok, logp, t, None, p, None, "odd values")


def test_edges_of_u(cuda_device):
    lg = torch.zeros(6, 100, device="cuda")
    lg[:, 3:] = -200.0  # weight 0
    u = f32([0.0, 1.0, 5.0, -1.0, float("nan"), 1 - 2 ** -24])
    tok, _ = na.sample(lg, u)
    assert tok.tolist() == [0, 2, 2, 0, 0, 2]


def test_frequencies(cuda_device):
    """An even grid of u gives each token its share of the grid to within one point."""
    n, V = 4096, 50
    lg = (torch.randn(1, V, generator=torch.Generator().manual_seed(2)) * 1.5).cuda().expand(n, V).contiguous()
    u = (torch.arange(n, device="cuda").float() + 0.5) / n
    tok, logp = na.sample(lg, u)
    share = torch.bincount(tok.long(), minlength=V).double() / n
    assert (share - lg[0].double().softmax(0)).abs().max() <= 1.0 / n + 1e-9
    assert (logp.double().exp() - lg[0].double().softmax(0)[tok.long()]).abs().max() < 1e-6
    assert (tok[1:] >= tok[:-1]).all()


def test_runs_are_identical_and_captured(cuda_device):
    lg, u = make(40, 100003, torch.float32, seed=4)
    p, k = f32([0.95] * 40), i32([0, 50] * 20)
    a = na.sample(lg, u, top_p=p, top_k=k)
    st = torch.cuda.Stream()
    tok, logp = torch.empty_like(a[0]), torch.empty_like(a[1])
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st):
        na.sample(lg, u, top_p=p, top_k=k, out_tok=tok, out_logp=logp, stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(a[0], tok) and torch.equal(a[1], logp)
    check(lg, u, *a, None, k, p, None)
