"""Cases and plain forms of the sampling decoder's operators.

Three operators that a program runs when it draws translations instead of searching them:

  paged   attention of a chunk of new target tokens over a paged key/value cache: the new rows are written
          into their pages and every new token attends to the positions up to its own;
  cross   cross-attention of many target rows to encoder states of another length, with a key mask;
  sample  one token for each row of logits by temperature, top-k, top-p and min-p, from given uniform numbers.

Where `own` is false, `run` computes them with elementary torch operations; where it is true it calls the
library through its Python binding.
"""
import math
import os
import random
import sys

import torch

own = False

_DT = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_GROUP = 1 << 29  # values of one temporary of the plain forms
_state = {}


def _library():
    if "na" not in _state:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bare-metal-nllb_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import nllb_attn
        _state["na"] = nllb_attn
    return _state["na"]


def _context(device):
    """The context of a GPU, on torch's current stream there."""
    na = _library()
    if device not in _state:
        _state[device] = [na.Context(device, n_layers=0, max_sentences=0), None]
    held, stream = _state[device], na.current_stream(device)
    if held[1] != stream:
        held[0].set_stream(stream)
        held[1] = stream
    return held[0]


# ---- cases ---------------------------------------------------------------------------------------------------


def listed():
    return [
        # one sentence, one new token after 99 cached ones, 16 heads of 64 in fp32: the latency of a decoder step
        dict(name="paged_one_token", op="paged", dtype="float32", n_seq=1, q_lo=1, q_hi=1, past_lo=99, past_hi=99,
             heads=16, kv_heads=16, dim=64, page=16),
        # a serving batch: one token for each of 64 sequences of very different lengths, four query heads to a key head
        dict(name="paged_batch_tokens", op="paged", dtype="bfloat16", n_seq=64, q_lo=1, q_hi=1, past_lo=200,
             past_hi=8191, heads=16, kv_heads=4, dim=128, page=16),
        # one token far into a long document, two key heads only: the work has to be split over the keys
        dict(name="paged_long_token", op="paged", dtype="float16", n_seq=1, q_lo=1, q_hi=1, past_lo=99990,
             past_hi=99990, heads=16, kv_heads=2, dim=64, page=48),
        # forced target prefixes of up to 132 tokens for 64 sentences, nothing cached before: the engine's own sizes
        dict(name="paged_prefix", op="paged", dtype="float32", n_seq=64, q_lo=1, q_hi=132, past_lo=0, past_hi=0,
             heads=16, kv_heads=16, dim=64, page=16),
        # chunks of a long prompt for 8 sequences, each behind a cache of its own length
        dict(name="paged_chunks", op="paged", dtype="bfloat16", n_seq=8, q_lo=500, q_hi=1024, past_lo=0, past_hi=7000,
             heads=32, kv_heads=8, dim=64, page=64),
        # one short sentence scored against its source: 21 target rows, 74 source rows
        dict(name="cross_sentence", op="cross", dtype="float32", n_seq=1, q_lo=21, q_hi=21, kv_lo=74, kv_hi=74,
             heads=16, kv_heads=16, dim=64, mask=0.0),
        # one decoder step of 256 sequences over memories of 18 to 512 rows held in 16 bits
        dict(name="cross_tokens", op="cross", dtype="bfloat16", n_seq=256, q_lo=1, q_hi=1, kv_lo=18, kv_hi=512,
             heads=16, kv_heads=16, dim=64, mask=0.0),
        # target sides of up to 132 tokens of 128 sentences scored against sources of 18 to 130 rows
        dict(name="cross_batch", op="cross", dtype="float32", n_seq=128, q_lo=9, q_hi=132, kv_lo=18, kv_hi=130,
             heads=16, kv_heads=16, dim=64, mask=0.0),
        # long documents, heads of 128, a tenth of the source rows masked out
        dict(name="cross_documents", op="cross", dtype="bfloat16", n_seq=4, q_lo=1500, q_hi=2048, kv_lo=3500,
             kv_hi=4096, heads=16, kv_heads=16, dim=128, mask=0.1),
        # one row of the vocabulary: the latency of a single drawn token
        dict(name="sample_row", op="sample", dtype="float32", rows=1, vocab=256206, temperature=0.8, top_k=50,
             top_p=0.95, min_p=0.0),
        # 64 rows, nucleus sampling alone, logits in 16 bits
        dict(name="sample_nucleus", op="sample", dtype="bfloat16", rows=64, vocab=256206, temperature=1.0, top_k=0,
             top_p=0.9, min_p=0.0),
        # the engine's largest share of rows, each with settings of its own (top-k, top-p, min-p, none, greedy)
        dict(name="sample_mixed", op="sample", dtype="float32", rows=512, vocab=256206, temperature=-1.0, top_k=-1,
             top_p=-1.0, min_p=-1.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["paged", "paged", "cross", "cross", "sample"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "sample":
        mixed = rng.random() < 0.4
        return dict(op="sample", dtype=dtype, rows=_log_int(rng, 1, 512), vocab=_log_int(rng, 1000, 256206),
                    temperature=-1.0 if mixed else rng.choice([0.5, 0.8, 1.0, 1.5]),
                    top_k=-1 if mixed else rng.choice([0, 1, 8, 50, 1000]),
                    top_p=-1.0 if mixed else rng.choice([1.0, 0.9, 0.95, 0.5]),
                    min_p=-1.0 if mixed else rng.choice([0.0, 0.0, 0.05, 0.1]))
    kv_heads, group = rng.choice([(16, 1), (16, 1), (4, 4), (8, 4), (2, 8), (1, 12), (3, 5)])
    heads, dim = kv_heads * group, rng.choice([64, 64, 128])
    one = rng.random() < 0.4
    n_seq = _log_int(rng, 1, 256 if one else 64)
    # no dearer than the largest listed cases: 2^27 16-bit values of keys, 4e10 products (fp32 takes three of them)
    wide = dtype == "float32"
    values = 2 ** 27 // (2 if wide else 1) // (n_seq * kv_heads * dim)
    pairs = 4 * 10 ** 10 // (3 if wide else 1) // (n_seq * heads * dim)
    most = max(2, 2 ** 26 // (2 if wide else 1) // (n_seq * heads * dim))
    if op == "paged":
        q_hi = 1 if one else _log_int(rng, 2, min(1024, most))
        cap = min(100000, values, pairs // q_hi) - q_hi
        past_hi = 0 if cap < 16 or rng.random() < 0.15 else _log_int(rng, 1, cap)
        return dict(op="paged", dtype=dtype, n_seq=n_seq, q_lo=max(1, q_hi // rng.choice([1, 2, 8])), q_hi=q_hi,
                    past_lo=past_hi // rng.choice([1, 3, 20]), past_hi=past_hi, heads=heads, kv_heads=kv_heads,
                    dim=dim, page=rng.choice([16, 16, 32, 64, 128, 1, 7, 48]))
    q_hi = 1 if one else _log_int(rng, 2, min(2048, most))
    kv_hi = _log_int(rng, 2, max(3, min(8192, values, pairs // q_hi)))
    return dict(op="cross", dtype=dtype, n_seq=n_seq, q_lo=max(1, q_hi // rng.choice([1, 2, 8])), q_hi=q_hi,
                kv_lo=max(1, kv_hi // rng.choice([1, 2, 8])), kv_hi=kv_hi, heads=heads, kv_heads=kv_heads, dim=dim,
                mask=rng.choice([0.0, 0.0, 0.1, 0.5]))


def _lengths(case):
    """The query and key lengths of each sequence: the case's own, the same for every seed."""
    r = random.Random(case["n_seq"] * 1000003 + case["q_hi"] * 1009 + case["dim"])
    if case["op"] == "paged":
        q = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["n_seq"])]
        return q, [n + r.randint(case["past_lo"], case["past_hi"]) for n in q]
    return ([r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["n_seq"])],
            [r.randint(case["kv_lo"], case["kv_hi"]) for _ in range(case["n_seq"])])


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * 28, "flops": 4 * n}
    q, kv = _lengths(case)
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    rows, keys = sum(q), sum(kv)
    if case["op"] == "paged":
        pairs = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(q, kv))
        # queries and outputs; cached and new rows read, new rows written; lengths and page numbers
        moved = 2 * rows * h * d * size + 2 * keys * g * d * size + 2 * rows * g * d * size
        moved += 4 * (3 * len(q) + sum(-(-t // case["page"]) for t in kv))
    else:
        pairs = sum(n * t for n, t in zip(q, kv))
        moved = 2 * rows * h * d * size + 2 * keys * g * d * size + 16 * len(q) + (keys if case["mask"] else 0)
    return {"bytes": moved, "flops": 4 * d * h * pairs}


# ---- inputs --------------------------------------------------------------------------------------------------


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(1000 + int(seed))
    dt = _DT[case["dtype"]]

    def normal(*shape, scale=1.0):
        x = torch.empty(shape, dtype=dt, device=dev)
        return x.normal_(0.0, scale, generator=gen)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    s = dict(case=case, device=dev.index)
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        ld = -(-vocab // 8) * 8  # rows start on 16 bytes, as the engine's logits do
        # a language model's logits: a broad bulk, a spread that differs from row to row, some tokens far ahead
        lg = torch.empty((rows, ld), dtype=torch.float32, device=dev).normal_(0.0, 1.0, generator=gen)
        lg *= torch.empty((rows, 1), device=dev).uniform_(1.0, 3.0, generator=gen)
        ahead = torch.randint(0, vocab, (rows, 24), device=dev, generator=gen)
        lg.scatter_add_(1, ahead, torch.empty((rows, 24), device=dev).exponential_(0.25, generator=gen) + 4.0)
        s["logits"] = lg.to(dt)[:, :vocab]
        r = random.Random(int(seed) * 7 + rows)

        def setting(key, choices, kind):
            v = case[key]
            v = [r.choice(choices) for _ in range(rows)] if v < 0 else [v] * rows
            return torch.tensor(v, dtype=kind, device=dev)

        s["temperature"] = setting("temperature", [0.0, 0.7, 0.9, 1.0, 1.3], torch.float32)
        s["top_k"] = setting("top_k", [0, 0, 1, 40, 500, 20000], torch.int32)
        s["top_p"] = setting("top_p", [1.0, 1.0, 0.6, 0.9, 0.98], torch.float32)
        s["min_p"] = setting("min_p", [0.0, 0.0, 0.02, 0.2], torch.float32)
        s["u"] = torch.rand((rows,), device=dev, generator=gen)
        if own:
            s["tokens"] = torch.empty((rows,), dtype=torch.int32, device=dev)
            s["logp"] = torch.empty((rows,), dtype=torch.float32, device=dev)
        return s

    q, kv = _lengths(case)
    rows, h, g, d = sum(q), case["heads"], case["kv_heads"], case["dim"]
    s["q"] = normal(rows, h, d, scale=2.0)  # scores with a deviation of 2 after the scaling by 1/sqrt(dim)
    s["q_len"], s["q_start"] = ints(q), ints([sum(q[:i]) for i in range(len(q))])
    s["kv_len"] = ints(kv)
    s["max_q"], s["max_kv"] = max(q), max(kv)
    if case["op"] == "paged":
        page = case["page"]
        need = [-(-t // page) for t in kv]
        pool = sum(need) + 3
        perm = torch.randperm(pool, device=dev, generator=gen).to(torch.int32)
        table = torch.full((len(kv), max(need)), -1, dtype=torch.int32, device=dev)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = perm[at:at + n]
            at += n
        s["table"] = table
        s["k_pages"], s["v_pages"] = normal(pool, page, g, d), normal(pool, page, g, d)
        s["k_new"], s["v_new"] = normal(rows, g, d), normal(rows, g, d)
    else:
        keys = sum(kv)
        s["k"], s["v"] = normal(keys, g, d), normal(keys, g, d)
        s["kv_start"] = ints([sum(kv[:i]) for i in range(len(kv))])
        s["mask"] = None
        if case["mask"]:
            s["mask"] = (torch.rand((keys,), device=dev, generator=gen) >= case["mask"]).to(torch.uint8)
    if own:
        ctx = _context(dev.index)
        s["out"] = torch.empty_like(s["q"])
        if case["op"] == "paged":
            s["args"] = ctx.paged_args(s["q"], s["k_pages"], s["v_pages"], s["table"], s["kv_len"], s["out"],
                                       k_new=s["k_new"], v_new=s["v_new"], q_start=s["q_start"], q_len=s["q_len"],
                                       max_q=s["max_q"], max_kv=s["max_kv"])
        else:
            s["args"] = ctx.cross_rows_args(s["q"], s["k"], s["v"], s["out"], q_start=s["q_start"], q_len=s["q_len"],
                                            kv_start=s["kv_start"], kv_len=s["kv_len"], max_q=s["max_q"],
                                            max_kv=s["max_kv"], key_mask=s["mask"])
    return s


# ---- one pass ------------------------------------------------------------------------------------------------


def run(s):
    op = s["case"]["op"]
    if own:
        if op == "paged":
            _context(s["device"]).paged(s["args"])
            return {"out": s["out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if op == "cross":
            _context(s["device"]).cross_rows(s["args"])
            return {"out": s["out"]}
        _library().sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                          min_p=s["min_p"], out_tok=s["tokens"], out_logp=s["logp"])
        return {"tokens": s["tokens"], "logp": s["logp"]}
    return {"paged": _paged, "cross": _cross, "sample": _sample}[op](s)


def _attend(q, k, v, seen):
    """q [B, Q, H, D], k and v [B, L, G, D], seen [B, Q, L] or [B, 1, L]: attention in 32 bits, no visible key
    gives zeros."""
    B, Q, H, D = q.shape
    L, G = k.shape[1], k.shape[2]
    q = q.float().view(B, Q, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, (H // G) * Q, D)
    scores = torch.matmul(q, k.float().permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(D)).view(B, G, H // G, Q, L)
    scores.masked_fill_(~seen.view(B, 1, 1, seen.shape[1], L), float("-inf"))
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    w = scores.sub_(top).exp_()
    total = w.sum(-1, keepdim=True)
    out = torch.matmul(w.view(B, G, (H // G) * Q, L), v.float().permute(0, 2, 1, 3)).view(B, G, H // G, Q, D)
    out = out / torch.where(total == 0, torch.ones_like(total), total)
    return out.permute(0, 3, 1, 2, 4).reshape(B, Q, H, D)


def _groups(n, size):
    step = max(1, min(n, _GROUP // max(1, size)))
    return [range(i, min(n, i + step)) for i in range(0, n, step)]


def _padded(x, start, length, most):
    """Rows [start, start + length) of each sequence as [B, most, ...], and which of them are there."""
    at = torch.arange(most, device=x.device)
    there = at[None, :] < length[:, None]
    rows = torch.where(there, start[:, None].long() + at, torch.zeros_like(at))
    return x[rows], there, rows


def _paged(s):
    c = s["case"]
    q, kp, vp, page = s["q"], s["k_pages"], s["v_pages"], c["page"]
    out = torch.empty_like(q)
    Q, L, n = s["max_q"], s["max_kv"], c["n_seq"]
    at, keys = torch.arange(Q, device=q.device), torch.arange(L, device=q.device)
    for grp in _groups(n, L * max(c["kv_heads"] * c["dim"], c["heads"] * Q)):
        sl = slice(grp.start, grp.stop)
        ql, kl, table = s["q_len"][sl], s["kv_len"][sl], s["table"][sl].long()
        qq, there, rows = _padded(q, s["q_start"][sl], ql, Q)
        pos = (kl - ql)[:, None] + at
        slot = torch.where(there, table.gather(1, (pos // page).clamp(0, table.shape[1] - 1).long()), -1)
        kp[slot[there], (pos % page)[there]] = s["k_new"][rows[there]]
        vp[slot[there], (pos % page)[there]] = s["v_new"][rows[there]]
        where = table[:, keys // page].clamp(min=0)
        k, v = kp[where, keys % page], vp[where, keys % page]
        alive = keys[None, :] < kl[:, None]
        v = v.masked_fill(~alive[:, :, None, None], 0)
        o = _attend(qq, k, v, (keys <= pos[:, :, None]) & alive[:, None, :])
        out[rows[there]] = o[there].to(out.dtype)
    return {"out": out, "k_pages": kp, "v_pages": vp}


def _cross(s):
    c = s["case"]
    q = s["q"]
    out = torch.empty_like(q)
    Q, L = s["max_q"], s["max_kv"]
    for grp in _groups(c["n_seq"], L * max(c["kv_heads"] * c["dim"], c["heads"] * Q)):
        sl = slice(grp.start, grp.stop)
        qq, there, rows = _padded(q, s["q_start"][sl], s["q_len"][sl], Q)
        k, alive, at = _padded(s["k"], s["kv_start"][sl], s["kv_len"][sl], L)
        v = s["v"][at]
        if s["mask"] is not None:
            alive = alive & (s["mask"][at] != 0)
        v = v.masked_fill(~alive[:, :, None, None], 0)
        o = _attend(qq, k, v, alive[:, None, :])
        out[rows[there]] = o[there].to(out.dtype)
    return {"out": out}


_LEAST = 2.0 ** -45  # a token of less weight beside the likeliest one is never drawn


def _sample(s):
    """Weights and their running sums in 64 bits: a token's border lies anywhere between its neighbours'."""
    rows, vocab = s["logits"].shape
    toks, lps = [], []
    for grp in _groups(rows, vocab * 4):
        sl = slice(grp.start, grp.stop)
        lg = s["logits"][sl].float()
        lg = torch.where(torch.isnan(lg), torch.full_like(lg, float("-inf")), lg)
        t = s["temperature"][sl].double()[:, None]
        greedy = t == 0
        lv, order = torch.sort(lg, dim=1, descending=True, stable=True)
        x = (lv.double() - lv[:, :1].double()) / torch.where(greedy, torch.ones_like(t), t)
        x = torch.where(lv == lv[:, :1], torch.zeros_like(x), x)
        w = x.exp()
        w = torch.where(w < _LEAST, torch.zeros_like(w), w)
        at = torch.arange(vocab, device=lg.device)[None, :]
        k = s["top_k"][sl].long()[:, None]
        k = torch.where((k <= 0) | (k > vocab), torch.full_like(k, vocab), k)
        k = torch.where(greedy, torch.ones_like(k), k)
        w = w * (at < k)
        p = s["top_p"][sl].double()[:, None]
        before = w.cumsum(1) - w
        keep = (at == 0) | (p >= 1) | (before < p * w.sum(1, keepdim=True))
        keep &= (at == 0) | (w >= s["min_p"][sl].double()[:, None])
        w = w * keep
        del before, keep
        w = torch.zeros_like(w).scatter_(1, order, w)
        x = torch.zeros_like(x).scatter_(1, order, x)
        total = w.sum(1, keepdim=True)
        tok = ((w.cumsum(1) > s["u"][sl].double()[:, None] * total) & (w > 0)).to(torch.uint8).argmax(1, keepdim=True)
        toks.append(tok[:, 0].to(torch.int32))
        lps.append((x.gather(1, tok) - total.log())[:, 0].float())
    return {"tokens": torch.cat(toks), "logp": torch.cat(lps)}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------


def exact(case, seed):
    plain = own
    globals()["own"] = False  # the inputs alone
    try:
        s = prepare(case, seed)
    finally:
        globals()["own"] = plain
    return _exact_sample(s) if case["op"] == "sample" else _exact_attention(s)


def _exact_attention(s):
    c = s["case"]
    h, g, d = c["heads"], c["kv_heads"], c["dim"]
    ql, kl = _lengths(c)
    out = torch.empty_like(s["q"], dtype=torch.float64)
    paged = c["op"] == "paged"
    row = key = 0
    for i, (n, t) in enumerate(zip(ql, kl)):
        if paged:
            pages = s["table"][i, :-(-t // c["page"])].long()
            k = s["k_pages"][pages].reshape(-1, g, d)[:t].clone()
            v = s["v_pages"][pages].reshape(-1, g, d)[:t].clone()
            k[t - n:], v[t - n:] = s["k_new"][row:row + n], s["v_new"][row:row + n]
        else:
            k, v = s["k"][key:key + t], s["v"][key:key + t]
            if s["mask"] is not None:
                left = s["mask"][key:key + t].nonzero()[:, 0]
                k, v = k[left], v[left]
            key += t
        for j in range(h):
            kk, vv = k[:, j * g // h].double(), v[:, j * g // h].double()
            if not len(kk):
                out[row:row + n, j] = 0
                continue
            sc = s["q"][row:row + n, j].double() @ kk.T / math.sqrt(d)
            if paged:
                sc = sc + torch.full_like(sc, float("-inf")).triu_(t - n + 1)
            e = torch.exp(sc - sc.max(1, keepdim=True)[0])
            out[row:row + n, j] = (e @ vv) / e.sum(1, keepdim=True)
        row += n
    if not paged:
        return {"out": out}
    return {"out": out, "k_pages": None, "v_pages": None}  # copies, not computed numbers


def _exact_sample(s):
    rows, vocab = s["logits"].shape
    toks, lps = [], []
    for r in range(rows):
        lg = s["logits"][r].double()
        lg[torch.isnan(lg)] = float("-inf")
        t, k, p, m, u = (float(s[n][r]) for n in ("temperature", "top_k", "top_p", "min_p", "u"))
        best = float(lg.max())
        if t == 0:
            toks.append(int((lg == best).nonzero()[0, 0]))
            lps.append(0.0)
            continue
        w = torch.exp((lg - best) / t)
        w[lg == best] = 1.0
        w[w < _LEAST] = 0.0
        idx = torch.argsort(-lg, stable=True)
        if 0 < k < vocab:
            idx = idx[:int(k)]
        if p < 1:
            run_sum = torch.cumsum(w[idx], 0)
            # the shortest run whose sum reaches p of the whole
            n = int((run_sum < p * run_sum[-1]).sum()) + 1
            idx = idx[:n]
        idx = idx[:max(1, int((w[idx] >= m).sum()))]
        idx = torch.sort(idx)[0]
        idx = idx[w[idx] > 0]
        c = torch.cumsum(w[idx], 0)
        j = int((c <= u * c[-1]).sum())
        tok = int(idx[min(j, len(idx) - 1)])
        toks.append(tok)
        lps.append(float(lg[tok] - best) / t - math.log(float(c[-1])))
    return {"tokens": torch.tensor(toks, dtype=torch.int32), "logp": torch.tensor(lps, dtype=torch.float64)}
