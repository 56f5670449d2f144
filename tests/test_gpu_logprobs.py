"""nllb_logprobs on the GPU against the definition in 64 bits.

Tolerances, derived from the arithmetic and set before the first run.  With u = 2^-24, d_i = max l - l_i, E[.] the mean
under the row's softmax and n the vocabulary: the scaled difference y_i is rounded once (u d_i) and its factor log2(e)
carries a relative 2 u, which scales every difference alike (2 u d_t, and 2 u E[d] through log Z); a weight's exponential is
off by 4 u; a thread adds n / 512 weights in two chains, and 5 + 4 + 4 joins follow with two roundings each, so log Z is
off by (n / 1024 + 64) u at most; its logarithm and the last products add 4 u of their sizes.  The entropy's second sum
has terms w d with the errors of w times d, so E[d^2] u, 4 u E[d] and the chain's (n / 1024 + 64) u E[d]."""
import math

import pytest
import torch

import nllb_attn as na

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def expected(row, target, n):
    """(logp, entropy, tokens, their logp, tolerance of logp per token, of the entropy) of a row of finite logits or -inf."""
    x = row.double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    chain = x.numel() / 1024 + 64
    if not (x > -math.inf).any():
        p = torch.full_like(x, -math.inf)
        entropy, tol, tol_h = 0.0, torch.zeros_like(x), 0.0
    elif x.max() == math.inf:
        same = x == math.inf
        p = torch.where(same, -math.log(int(same.sum())), -math.inf)
        entropy, tol, tol_h = math.log(int(same.sum())), torch.full_like(x, 16 * U * math.log(x.numel() + 2)), 16 * U * math.log(x.numel() + 2)
    else:
        d = x.max() - x
        w = torch.exp(-d)
        z = w.sum()
        p = -d - z.log()
        w = w / z
        dd = torch.where(w > 0, d, 0.0)
        e1, e2, log_z = float((w * dd).sum()), float((w * dd * dd).sum()), float(z.log())
        entropy = log_z + e1
        tol = U * (chain + 16 + 4 * e1 + 8 * log_z + 8 * torch.where(d < math.inf, d, 0.0))
        tol_h = U * ((chain + 16) * (1 + e1) + 4 * e2 + 8 * e1 + 8 * log_z)
    order = torch.argsort(-x, stable=True)[:n]
    order = order[x[order] > -math.inf]
    return p, entropy, order, tol, tol_h


def check(logits, target, out, n, what=""):
    logp, entropy, tok, top = out
    rows, vocab = logits.shape
    for r in range(rows):
        t = None if target is None else int(target[r])
        if t is not None and t < 0:
            assert float(logp[r]) == 0 and float(entropy[r]) == 0, f"{what} padding {r}"
            if n:
                assert (tok[r] == -1).all() and (top[r] == -math.inf).all(), f"{what} padding {r}"
            continue
        p, h, order, tol, tol_h = expected(logits[r].cpu(), t, n)
        if t is not None:
            got = float(logp[r])
            want = float(p[t]) if t < vocab else -math.inf
            assert got == want or abs(got - want) <= float(tol[t]), f"{what} row {r}: logp {got} for {want}, {float(tol[t])}"
        if entropy is not None:
            assert abs(float(entropy[r]) - h) <= tol_h, f"{what} row {r}: entropy {float(entropy[r])} for {h}, {tol_h}"
        if n:
            k = len(order)
            assert tok[r].cpu().tolist() == order.tolist() + [-1] * (n - k), f"{what} row {r}: tokens"
            got = top[r].double().cpu()
            assert (got[k:] == -math.inf).all(), f"{what} row {r}"
            got, want = got[:k], p[order]
            assert ((got == want) | ((got - want).abs() <= tol[order])).all(), f"{what} row {r}: logp of tokens"


def logits_of(rows, vocab, dtype, seed, ld=None):
    """A language model's: a bulk, and some tokens far ahead."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, ld or vocab, generator=g) * (1 + 2 * torch.rand(rows, 1, generator=g))
    at = torch.randint(0, vocab, (rows, 6), generator=g)
    x.scatter_add_(1, at, 4 + 4 * torch.rand(rows, 6, generator=g))
    return x.to(dtype).cuda()[:, :vocab], at[:, 0].to(torch.int32).cuda()


def run(logits, target, n, what="", **kw):
    out = na.logprobs(logits, target, top_n=n, **kw)
    torch.cuda.synchronize()
    check(logits, target, out, n, what)
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,pad,n", [
    (1, 1, 0, 1), (3, 2, 0, 5), (2, 7, 1, 8), (5, 31, 0, 32), (4, 33, 2, 3), (7, 997, 3, 20), (2, 4096, 0, 0), (3, 8195, 5, 32),
    (1, 256206, 0, 8), (2, 256206, 2, 32), (9, 100003, 0, 1), (300, 2001, 0, 5), (700, 515, 1, 4)])
def test_sizes(cuda_device, dtype, rows, vocab, pad, n):
    lg, t = logits_of(rows, vocab, dtype, rows * 7 + vocab, vocab + pad)
    run(lg, t, n)


@pytest.mark.parametrize("rows", [1, 20, 330])
def test_rows_of_every_alignment(cuda_device, rows):
    """A contiguous matrix whose rows start anywhere, and a matrix that starts anywhere."""
    for dtype in TYPES:
        for off in (0, 1, 3, 7):
            vocab = 20011
            lg, t = logits_of(1, rows * vocab + off, dtype, off)
            lg = lg[0, off:].view(rows, vocab)
            run(lg, torch.arange(rows, dtype=torch.int32, device="cuda") * 60 % vocab, 16, f"{dtype} {off}")


def shaped(kind, vocab, dtype):
    i = torch.arange(vocab)
    x = {
        "equal": torch.zeros(vocab),
        "equal and a zero of either sign": torch.where(i % 3 == 1, -0.0, 0.0),
        "rising": i / vocab * 8,
        "falling": -i / vocab * 8,
        # what one thread reads comes first as a whole: vectors that lie 512 apart
        "one stripe": torch.where(i // 8 % 512 == 5, 9.0, 0.0) + i / vocab,
        "one stripe of 32 bits": torch.where(i // 4 % 512 == 77, 9.0, 0.0) - i / vocab,
        "few values": (i * 7919 % 11).float(),
        "the last ones": torch.where(i >= vocab - 3, 5.0, i % 13 / 13),
        "the first ones": torch.where(i < 3, 5.0, i % 13 / 13),
        "one is all": torch.where(i == vocab // 2, 60.0, -20.0),
        "masked": torch.where(i % 5 == 0, i % 101 / 10, -math.inf),
        "two left": torch.where((i == 1) | (i == vocab - 1), 1.0, -math.inf),
        "nothing left": torch.full((vocab,), -math.inf),
        "NaN": torch.where(i % 4 == 0, math.nan, i % 101 / 10),
        "all NaN": torch.full((vocab,), math.nan),
        "infinite": torch.where(i % 1000 == 3, math.inf, i % 101 / 10),
        "infinite and NaN": torch.where(i % 1000 == 3, math.inf, torch.where(i % 2 == 0, math.nan, -math.inf)),
    }[kind]
    return x.float().to(dtype)


KINDS = ["equal", "equal and a zero of either sign", "rising", "falling", "one stripe", "one stripe of 32 bits", "few values",
         "the last ones", "the first ones", "one is all", "masked", "two left", "nothing left", "NaN", "all NaN", "infinite",
         "infinite and NaN"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", KINDS)
def test_shapes_of_rows(cuda_device, dtype, kind):
    for rows, vocab in ((1, 50021), (1, 3), (40, 20011), (400, 6007)):
        x = shaped(kind, vocab, dtype).cuda()
        if kind == "infinite" and vocab == 3:
            continue
        lg = x.repeat(rows, 1)
        t = torch.full((rows,), vocab // 2, dtype=torch.int32, device="cuda")
        t[0] = vocab - 1
        few = slice(0, 3)  # (the others are the same row, and start at the same place of 16 bytes every `period` rows)
        period = 16 // lg.element_size()
        out = na.logprobs(lg, t, top_n=32)
        torch.cuda.synchronize()
        check(lg[few], t[few], [o[few] for o in out], 32, kind)
        assert all((o[1 + period:] == o[1:-period]).all() for o in out[1:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_of_the_types_ends(cuda_device, dtype):
    """The largest share the weight, and a row of the type's lowest value is an even one."""
    least = torch.finfo(dtype).min
    x = torch.full((4, 9001), least, dtype=dtype, device="cuda")
    x[1, 100:140] = 1.0
    x[2, 7:9] = torch.finfo(dtype).max
    x[3, 17] = -1e38
    t = torch.tensor([5, 120, 8, 17], dtype=torch.int32, device="cuda")
    logp, h, tok, top = na.logprobs(x, t, top_n=3)
    torch.cuda.synchronize()
    for got, want in zip(logp.tolist(), (-math.log(9001), -math.log(40), -math.log(2), 0.0)):
        assert abs(got - want) <= 128 * U
    for got, want in zip(h.tolist(), (math.log(9001), math.log(40), math.log(2), 0.0)):
        assert abs(got - want) <= 128 * U
    assert tok.tolist() == [[0, 1, 2], [100, 101, 102], [7, 8, 0], [17, 0, 1]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", [-1e4, -1e9, -1e30])
def test_masked_by_a_low_value(cuda_device, dtype, mask):
    """Rows masked by a low value in long runs, so that whole threads see nothing else, and rows that are nothing else."""
    mask = max(mask, torch.finfo(dtype).min)
    lg, t = logits_of(4, 60013, dtype, 9)
    lg[0, 40000:] = mask
    lg[1, 300:] = mask
    lg[2, :] = mask
    t[0], t[1], t[2] = 50000, 7, 60012
    run(lg, t, 32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gap", [4.0, 12.0, 20.0, 40.0])
@pytest.mark.parametrize("base", [0.0, 37.7])
def test_dominated_rows(cuda_device, dtype, gap, base):
    """One token far ahead of very many: what is left to the others is small, and as accurate relative to its size.  Each of
    their weights is off by 4 u, and by u of its difference and 2 u of it by log2(e)'s rounding, their sums by the chain's
    (n / 1024 + 64) u; the logarithm of 1 + z and the quotient add 8 u."""
    g = torch.Generator().manual_seed(int(gap))
    for rows, vocab in ((1, 256206), (3, 50021), (200, 3001)):
        x = base + torch.rand(rows, vocab, generator=g)
        x[:, vocab // 3] = base + 1 + gap
        lg = x.to(dtype).cuda()
        t = torch.full((rows,), vocab // 3, dtype=torch.int32, device="cuda")
        logp, h, _, _ = na.logprobs(lg, t)
        d = lg[:, vocab // 3:vocab // 3 + 1].double() - lg.double()
        w = torch.exp(-d)
        w[:, vocab // 3] = 0
        z = w.sum(1)
        want = torch.log1p(z)
        want_h = want + (w * d).sum(1) / (1 + z)
        rel = U * (vocab / 1024 + 64 + 3 * (gap + 1) + 16)
        assert ((-logp.double() / want - 1).abs() <= rel).all(), f"{rows} x {vocab}: logp"
        assert ((h.double() / want_h - 1).abs() <= 2 * rel).all(), f"{rows} x {vocab}: entropy"


@pytest.mark.parametrize("top", [1e6, 1e8, 2.0 ** 27 + 16, 2.0 ** 28, 1e12, 1e37])
def test_large_logits(cuda_device, top):
    """A few of the largest, the next ones a step of the type lower, and a bulk far below; of either sign."""
    for sign in (1, -1):
        x = torch.zeros(3, 4099) if sign > 0 else torch.full((3, 4099), -3e38)
        x[:, 5:9] = sign * top
        step = torch.nextafter(x[0, 5], torch.tensor(-math.inf))
        x[1, 1000:1003] = step
        x = x.cuda()
        run(x, torch.tensor([5, 1001, 0], dtype=torch.int32, device="cuda"), 12, f"{sign} {top}")


def test_padding_and_foreign_targets(cuda_device):
    lg, t = logits_of(6, 5003, torch.float32, 3)
    lg[1] = math.nan
    t[1], t[2], t[4] = -1, 5003, -(2 ** 31)
    t[5] = 2 ** 31 - 1
    run(lg, t, 4)
    run(lg, None, 4)


def test_only_what_is_asked_for(cuda_device):
    lg, t = logits_of(3, 777, torch.float16, 4)
    logp, h, tok, top = run(lg, t, 0)
    assert tok is None and top is None
    only = na.logprobs(lg, t, entropy=False)
    assert only[1] is None and (only[0] == logp).all()
    assert na.logprobs(lg)[0] is None and (na.logprobs(lg)[1] == h).all()
    alone = na.logprobs(lg, top_n=2, entropy=False)
    assert alone[0] is None and alone[1] is None
    check(lg, None, (None, None, *alone[2:]), 2)


def test_same_result_in_any_company(cuda_device):
    """A row's result does not depend on the rows beside it while as many CTAs share it, nor on the run."""
    whole, t = logits_of(8, 30016, torch.bfloat16, 5)  # (every row starts on 16 bytes)
    t %= 30011
    a = run(whole[:, :30011], t, 9)
    b = run(whole.flip(0)[:, :30011], t.flip(0), 9)
    assert all((x == y.flip(0)).all() for x, y in zip(a, b))


def test_on_a_stream_and_captured(cuda_device):
    lg, t = logits_of(5, 70001, torch.float32, 6)
    late = torch.full_like(lg, -1.0)
    na.logprobs(late, t, top_n=5)  # (a kernel's first launch may wait for the device)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        torch.cuda._sleep(20_000_000)
        late.copy_(lg)
        out = na.logprobs(late, t, top_n=5)
        kept = [o.clone() for o in out]
    st.synchronize()
    check(lg, t, kept, 5, "on the current stream")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        na.logprobs(late, t, top_n=5, out_logp=out[0], out_entropy=out[1], out_top_tok=out[2], out_top_logp=out[3])
    lg, _ = logits_of(5, 70001, torch.float32, 7)
    late.copy_(lg)
    g.replay()
    torch.cuda.synchronize()
    check(lg, t, out, 5, "replayed")


def test_beside_the_search(cuda_device):
    """The tokens of nllb_logsoftmax_topk, with its log-probabilities."""
    lg, t = logits_of(6, 20011, torch.float32, 8)
    tok, lp = na.logsoftmax_topk(lg.contiguous(), 8)
    _, _, top, logp = na.logprobs(lg, t, top_n=8)
    assert (tok == top).all() and (lp - logp).abs().max() < 1e-4
