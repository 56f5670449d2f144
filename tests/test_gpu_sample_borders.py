"""nllb_sample where its internal steps, its types' ends and its settings' ends meet the logits: against the definition
in 64 bits (the same reference as test_gpu_sample.py).

The kernel places logits on a scale of 2048 steps of 33/2048 temperatures.  The inputs here lie on the edges of those
steps, a few units of fp32 to either side, alone and by the thousand.  Tokens have to be equal; `border_margin` keeps
the shares that top-p asks for away from a border by more than the kernel's units can move it (2^19 halves of 2^-44
are below 2e-8 of the largest weight), and `check` does so for u."""
import numpy as np
import pytest
import torch

import nllb_attn as na
from test_gpu_sample import LEAST, check, f32, i32

pytestmark = pytest.mark.gpu

STEP = 33.0 / 2048.0


def border_margin(lg, t, k, p):
    """Distance, in units of the largest weight, of top-p's share from the nearest sum where the cut would move."""
    lg = lg.astype(np.float64)
    x = (lg - lg.max()) / t
    w = np.sort(np.where(np.exp(x) < LEAST, 0, np.exp(x)))[::-1]
    if 0 < k < len(w):
        w = w[:k]
    c = np.cumsum(w)
    return np.abs(c - p * c[-1]).min()


def share(lg, t, k, first):
    """The first share at or above `first` that is not near a border."""
    for i in range(2000):
        p = np.float32(first + i * 1.7e-4)
        if border_margin(lg, t, k, float(p)) > 1e-6:
            return float(p)
    raise AssertionError("no such share")


def edge_logits(t, steps):
    """Logits half-way between steps below 0, with their neighbours in fp32."""
    e = np.float32(-(np.asarray(steps) + 0.5) * STEP * t)
    out = [e]
    lo = hi = e
    for _ in range(3):
        lo, hi = np.nextafter(lo, np.float32(-np.inf)), np.nextafter(hi, np.float32(0))
        out += [lo, hi]
    return np.stack(out, 1)  # [steps][7]


US = [0.03, 0.17, 0.31, 0.49, 0.62, 0.78, 0.93]


def run(rows, u, **kw):
    """rows [n][V] numpy, every setting a list; drawn three times, the answers have to be the same."""
    lg = torch.from_numpy(np.ascontiguousarray(rows)).cuda()
    names = dict(t="temperature", k="top_k", p="top_p", m="min_p")
    s = {names[n]: (i32 if n == "k" else f32)(v) for n, v in kw.items()}
    a = na.sample(lg, f32(u), **s)
    if "t" in kw:
        s["temperature"] = s["temperature"].clamp(max=2.0 ** 96)  # as the header says
    for _ in range(2):
        b = na.sample(lg, f32(u), **{**s, **({"temperature": f32(kw["t"])} if "t" in kw else {})})
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    check(lg, f32(u), *a, *[s.get(n) for n in ("temperature", "top_k", "top_p", "min_p")], what="borders")


def test_candidate_on_the_edge_of_the_last_step(cuda_device):
    """A logit half a step beyond the border's: counted or not, the candidates gathered are those counted."""
    row = np.full(1000, -np.inf, np.float32)
    row[127] = 0.0
    row[[0, 4, 8, 12, 16]] = -0.96680
    row[20] = -0.9748534560203552
    run(np.tile(row, (len(US), 1)), US, p=[0.6] * len(US), t=[1.0] * len(US))


@pytest.mark.parametrize("copies,vocab", [(1, 5127), (80, 5127), (200, 90003)], ids=["cluster", "cta", "streamed"])
def test_thousands_on_one_edge(cuda_device, copies, vocab):
    """5000 equal logits half-way between two steps, by top-p and by top-k, as one row and as many."""
    rows, t, k, p = [], [], [], []
    for s in (31, 60, 63, 300):
        for e in edge_logits(1.0, [s])[0][:3]:
            row = np.full(vocab, -np.inf, np.float32)
            row[7:7 + 3 * 5000:3 if vocab > 20000 else 1][:5000] = e
            row[vocab - 1] = 0.0
            for kk, first in ((0, 0.6), (3000, 0.4), (1700, 0.99)):
                rows.append(row)
                t.append(1.0)
                k.append(kk)
                p.append(share(row, 1.0, kk, first))
    n = len(rows)
    pick = range(0, n) if copies > 1 else [0, 4, 8, 9]
    if copies == 1:  # few rows: a cluster each
        for i in pick:
            run(rows[i][None], [0.37], t=[t[i]], k=[k[i]], p=[p[i]])
        return
    many = max(copies, n)
    at = [i % n for i in range(many)]
    u = [US[i % 7] for i in range(many)]
    run(np.stack([rows[i] for i in at]), u, t=[t[i] for i in at], k=[k[i] for i in at], p=[p[i] for i in at])


@pytest.mark.parametrize("t", [1.0, 0.7, 3.1])
@pytest.mark.parametrize("vocab", [14400, 90003])
def test_logits_on_every_edge(cuda_device, t, vocab):
    """All 2047 edges with three neighbours on each side, in any order; rows of 14400 from shared memory, 192 rows of
    90003 read in every pass."""
    rng = np.random.default_rng(vocab + int(10 * t))
    n = 24 if vocab < 20000 else 192
    edges = edge_logits(t, np.arange(2047)).ravel()
    rows = np.full((n, vocab), -np.inf, np.float32)
    k, p, u = [], [], []
    base = [rng.permutation(vocab)[:len(edges) + 1] for _ in range(3)]
    for r in range(n):
        at = base[r % 3]
        rows[r, at[:-1]] = edges
        rows[r, at[-1]] = 0.0
        k.append([0, 0, 224, 225, 231, 1000, 5000][r % 7])
        p.append([0.9, 0.5, 0.999, 1.0, 0.3][r % 5])
        u.append(US[(r * 3) % 7])
    cache = {}
    for r in range(n):
        key = (k[r], p[r])
        if p[r] < 1:
            if key not in cache:
                cache[key] = share(rows[r], float(np.float32(t)), k[r], p[r])
            p[r] = cache[key]
    run(rows, u, t=[t] * n, k=k, p=p)


def extreme_rows(vocab):
    """(logits, temperature) with masked tokens (-inf, NaN) at the lowest indices, and the weights of the others far
    above 0 whatever their size."""
    rng = np.random.default_rng(5)
    lowest, top = np.finfo(np.float32).min, np.finfo(np.float32).max
    sets = [
        (100.0, np.nextafter(np.float32(100), np.float32(0)), 1e-6),
        (20.0, np.nextafter(np.float32(20), np.float32(0)), 8e-8),
        (1.0, -4.0, 2e37),
        (1.0, -4.0, 1e38),
        (1.0e30, -1.0e30, 1e38),
        (top, lowest, 3.0e38),
        (2.0 ** 100, -2.0 ** 98, 9e36),
        (-2.0 ** 99, -2.0 ** 100, 2.0 ** 96),
        (-2.9e38, -3.0e38, 1e37),
        (np.nextafter(lowest, np.float32(0)), lowest, 1e32),
        (lowest, lowest, 1.0),
        (lowest, lowest, 1e38),
    ]
    rows, t = [], []
    for hi, lo, temp in sets:
        row = np.full(vocab, -np.inf, np.float32)
        row[1:300:3] = np.nan
        at = rng.permutation(np.arange(301, vocab))[:400]
        row[300], row[at[:150]], row[at[150:]] = hi, hi, lo
        rows.append(row)
        t.append(float(np.float32(temp)))
    return rows, t


@pytest.mark.parametrize("copies,vocab", [(1, 20011), (8, 3001), (16, 90003)], ids=["cluster", "cta", "streamed"])
def test_masked_tokens_weigh_nothing_at_any_temperature(cuda_device, copies, vocab):
    base, temps = extreme_rows(vocab)
    if copies == 1:
        for i, (row, t) in enumerate(zip(base, temps)):
            for kw in (dict(), dict(p=[0.77]), dict(k=[170], p=[0.9]), dict(m=[1e-3])):
                run(row[None], [[0.0, 0.999, 0.4][i % 3]], t=[t], **kw)
        return
    rows, t, u, k, p, m = [], [], [], [], [], []
    for c in range(copies):
        for row, temp in zip(base, temps):
            rows.append(row)
            t.append(temp)
            u.append([0.0, 0.9999, 0.37, 0.61][c % 4])
            k.append([0, 0, 170, 0][(c // 4) % 4])
            p.append([1.0, 0.77, 0.9, 1.0][(c // 4) % 4])
            m.append([0.0, 0.0, 0.0, 1e-3][(c // 4) % 4])
    run(np.stack(rows), u, t=t, k=k, p=p, m=m)


@pytest.mark.parametrize("rows,vocab", [(1, 20011), (9, 3001), (200, 90003)], ids=["cluster", "cta", "streamed"])
def test_min_p_of_one_keeps_the_largest_subnormal(cuda_device, rows, vocab):
    """The largest logit weighs 1 whatever its size, so a least weight of 1 keeps it and its equals."""
    for best, t in ((-1e-40, 2.0 ** -100), (-1e-45, 0.0009765625 * 2.0 ** -90), (0.0, 2.0 ** -100), (1e-40, 1e-30)):
        lg = np.full((rows, vocab), -1.0, np.float32)
        lg[:, 17::400] = best
        run(lg, [US[r % 7] for r in range(rows)], t=[t] * rows, m=[1.0] * rows)
