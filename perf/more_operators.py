"""Cases and plain forms of the operators around a decoder in 16 bits over a rolling paged cache.

Four operators that a program runs beside attention over the whole cache and the drawing of tokens:

  window    attention of a chunk of new target tokens over a paged cache where a token sees the last `window` positions
            and the first `sinks` ones (of a running translation: the tokens that name the language);
  append    new keys and values into a paged cache, queries and keys turned by their positions on the way;
  logprobs  log-probabilities of given tokens, the entropy of each row and its likeliest tokens;
  linear    a matrix product in 16 bits with bias, activation and residual.

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
        # one running translation, one new token after 5000, the last 1000 and the first 4 visible: a step's latency
        dict(name="window_one_token", op="window", dtype="float32", n_seq=1, q_lo=1, q_hi=1, past_lo=5000, past_hi=5000,
             heads=16, kv_heads=16, dim=64, page=16, window=1000, sinks=4),
        # a serving batch: one token for each of 64 sequences, some shorter than the window, most far longer
        dict(name="window_batch_tokens", op="window", dtype="bfloat16", n_seq=64, q_lo=1, q_hi=1, past_lo=500,
             past_hi=30000, heads=16, kv_heads=4, dim=128, page=16, window=4096, sinks=4),
        # chunks of long documents, each token of which sees the last 2000 and the first 16
        dict(name="window_chunks", op="window", dtype="float16", n_seq=8, q_lo=500, q_hi=1024, past_lo=0, past_hi=20000,
             heads=32, kv_heads=8, dim=64, page=64, window=2000, sinks=16),
        # one new token's queries turned, its key and value into the cache: the smallest call
        dict(name="append_one_token", op="append", dtype="float16", n_seq=1, q_lo=1, q_hi=1, past_lo=777, past_hi=777,
             heads=16, kv_heads=16, dim=64, page=16, rot=64, pairs="halves"),
        # a decoder step of 256 sequences of very different lengths
        dict(name="append_batch_tokens", op="append", dtype="bfloat16", n_seq=256, q_lo=1, q_hi=1, past_lo=10,
             past_hi=100000, heads=16, kv_heads=4, dim=128, page=16, rot=128, pairs="halves"),
        # whole prompts of 8 sequences, neighbouring values turned, the upper half of each head left as it is
        dict(name="append_prompts", op="append", dtype="bfloat16", n_seq=8, q_lo=1000, q_hi=4096, past_lo=0,
             past_hi=500, heads=32, kv_heads=8, dim=128, page=64, rot=64, pairs="neighbours"),
        # one row of the vocabulary, with the 8 likeliest tokens: what a step of a single translation reports
        dict(name="logprobs_row", op="logprobs", dtype="float32", rows=1, vocab=256206, pad=True, top=8),
        # forced decoding: 600 target tokens scored, nothing but their log-probabilities and the entropies
        dict(name="logprobs_score", op="logprobs", dtype="bfloat16", rows=600, vocab=256206, pad=True, top=0),
        # the tokens of 32 sentences, with 20 alternatives each, rows of a contiguous matrix (not on 16 bytes)
        dict(name="logprobs_alternatives", op="logprobs", dtype="float32", rows=1000, vocab=256206, pad=False, top=20),
        # the first feed-forward projection of a single token
        dict(name="linear_token", op="linear", dtype="bfloat16", m=1, n=4096, k=1024, act="relu", bias=True,
             residual=False, wide=False),
        # the vocabulary's logits of a decoder step of 64 rows, out in 32 bits
        dict(name="linear_logits", op="linear", dtype="bfloat16", m=64, n=256206, k=1024, act="none", bias=False,
             residual=False, wide=True),
        # the second feed-forward projection of a batch of prompts, added to the residual stream
        dict(name="linear_prompts", op="linear", dtype="float16", m=10000, n=1024, k=4096, act="none", bias=True,
             residual=True, wide=False),
    ]


_ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["window", "window", "append", "logprobs", "linear", "linear"])
    if op == "logprobs":
        # no dearer than the largest listed case: 4 GB / 4 of logits
        return dict(op=op, dtype=rng.choice(list(_DT)), rows=_log_int(rng, 1, 1000), vocab=_log_int(rng, 1000, 256206),
                    pad=rng.random() < 0.5, top=rng.choice([0, 1, 5, 8, 20, 32]))
    if op == "linear":
        m = _log_int(rng, 1, 10000)
        n = _log_int(rng, 64, min(256206, 2 ** 26 // max(m, 64)))
        k = _log_int(rng, 64, max(65, min(8192, 2 ** 35 // (m * n), 2 ** 27 // n)))
        if rng.random() < 0.6:  # widths of a model
            n, k = max(64, n // 64 * 64), max(64, k // 64 * 64)
        return dict(op=op, dtype=rng.choice(["float16", "bfloat16"]), m=m, n=n, k=k, act=rng.choice(_ACTS),
                    bias=rng.random() < 0.6, residual=rng.random() < 0.5, wide=rng.random() < 0.25)
    dtype = rng.choice(list(_DT))
    kv_heads, group = rng.choice([(16, 1), (4, 4), (8, 4), (2, 8), (1, 12), (3, 5)])
    heads, dim = kv_heads * group, rng.choice([64, 64, 128])
    one = rng.random() < 0.4
    n_seq = _log_int(rng, 1, 256 if one else 32)
    page = rng.choice([16, 16, 32, 64, 128, 1, 7, 48])
    wide = 2 if dtype == "float32" else 1
    if op == "append":
        most = 2 ** 26 // wide // (n_seq * (heads + kv_heads) * dim)
        q_hi = 1 if one else _log_int(rng, 2, max(2, min(4096, most)))
        past_hi = _log_int(rng, 1, 100000)
        return dict(op=op, dtype=dtype, n_seq=n_seq, q_lo=max(1, q_hi // rng.choice([1, 2, 8])), q_hi=q_hi,
                    past_lo=past_hi // rng.choice([1, 3, 20]), past_hi=past_hi, heads=heads, kv_heads=kv_heads, dim=dim,
                    page=page, rot=rng.choice([dim, dim, dim // 2, 0]), pairs=rng.choice(["halves", "neighbours"]))
    window, sinks = _log_int(rng, 1, 8192), rng.choice([0, 1, 4, 4, 16, 100])
    # no dearer than the largest listed cases: 2^27 16-bit values of keys, 2.4e10 products (fp32 takes three of them)
    span = window + sinks
    n_seq = max(1, min(n_seq, 2 ** 27 // wide // (kv_heads * dim * (span + 1)), 2 ** 26 // wide // (heads * dim)))
    most = min(24 * 10 ** 9 // (3 if wide == 2 else 1) // (n_seq * heads * dim * (span + 1)), 2 ** 24 // wide // (n_seq * heads * dim))
    q_hi = 1 if one or most < 2 else _log_int(rng, 2, min(1024, most))
    past_hi = min(30000, 2 ** 27 // wide // (n_seq * kv_heads * dim))
    past_hi = 0 if rng.random() < 0.15 else _log_int(rng, 1, max(2, past_hi))
    return dict(op=op, dtype=dtype, n_seq=n_seq, q_lo=max(1, q_hi // rng.choice([1, 2, 8])), q_hi=q_hi,
                past_lo=past_hi // rng.choice([1, 3, 20]), past_hi=past_hi, heads=heads, kv_heads=kv_heads, dim=dim,
                page=page, window=window, sinks=sinks)


def _lengths(case):
    """The new tokens and the whole length of each sequence: the case's own, the same for every seed."""
    r = random.Random(case["n_seq"] * 1000003 + case["q_hi"] * 1009 + case["dim"])
    q = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["n_seq"])]
    return q, [n + r.randint(case["past_lo"], case["past_hi"]) for n in q]


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    op = case["op"]
    if op == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (12 + 8 * case["top"]), "flops": 5 * n}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        out = 4 if case["wide"] else 2
        moved = 2 * (m * k + n * k) + out * m * n * (2 if case["residual"] else 1) + (2 * n if case["bias"] else 0)
        return {"bytes": moved, "flops": 2 * m * n * k}
    q, kv = _lengths(case)
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    rows = sum(q)
    if op == "append":
        pages = sum(-(-t // case["page"]) - (t - n) // case["page"] for n, t in zip(q, kv))
        moved = 2 * rows * (h + 2 * g) * d * size + 4 * (3 * len(q) + pages) + 2 * case["rot"]
        return {"bytes": moved, "flops": 3 * rows * (h + g) * case["rot"]}
    w, s = case["window"], case["sinks"]
    pairs = keys = 0
    for n, t in zip(q, kv):
        for p in range(t - n, t):
            lo = max(0, p - w + 1)
            pairs += p + 1 - lo + min(s, lo)
        lo = max(0, t - n - w + 1)
        keys += t - lo + min(s, lo)
    moved = 2 * rows * h * d * size + 2 * keys * g * d * size + 2 * rows * g * d * size
    moved += 4 * (3 * len(q) + keys // case["page"])
    return {"bytes": moved, "flops": 4 * d * h * pairs}


# ---- inputs --------------------------------------------------------------------------------------------------


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(1000 + int(seed))
    dt = _DT[case["dtype"]]

    def normal(*shape, scale=1.0, kind=dt):
        x = torch.empty(shape, dtype=kind, device=dev)
        return x.normal_(0.0, scale, generator=gen)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    s = dict(case=case, device=dev.index)
    if case["op"] == "logprobs":
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        ld = -(-vocab // 8) * 8 if case["pad"] else vocab
        # a language model's logits: a broad bulk, a spread that differs from row to row, some tokens far ahead
        lg = torch.empty((rows, ld), dtype=torch.float32, device=dev).normal_(0.0, 1.0, generator=gen)
        lg *= torch.empty((rows, 1), device=dev).uniform_(1.0, 3.0, generator=gen)
        ahead = torch.randint(0, vocab, (rows, 24), device=dev, generator=gen)
        lg.scatter_add_(1, ahead, torch.empty((rows, 24), device=dev).exponential_(0.25, generator=gen) + 4.0)
        s["logits"] = lg.to(dt)[:, :vocab]
        # given tokens: mostly likely ones, some from anywhere, a few rows of padding
        r = random.Random(int(seed) * 7 + rows)
        pick = torch.randint(0, 24, (rows, 1), device=dev, generator=gen)
        other = [-1 if rows > 8 and r.random() < 0.05 else r.randrange(vocab) if r.random() < 0.2 else -2 for _ in range(rows)]
        other = ints(other)
        s["target"] = torch.where(other > -2, other, ahead.gather(1, pick)[:, 0].to(torch.int32))
        if own:
            f32 = dict(dtype=torch.float32, device=dev)
            s["out"] = dict(out_logp=torch.empty(rows, **f32), out_entropy=torch.empty(rows, **f32))
            if top:
                s["out"]["out_top_tok"] = torch.empty((rows, top), dtype=torch.int32, device=dev)
                s["out"]["out_top_logp"] = torch.empty((rows, top), **f32)
        return s
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        ld = -(-k // 8) * 8  # rows start on 16 bytes
        out_dt = torch.float32 if case["wide"] else dt
        s["x"], s["w"] = normal(m, ld)[:, :k], normal(n, ld, scale=k ** -0.5)[:, :k]
        s["bias"] = normal(n) if case["bias"] else None
        s["residual"] = normal(m, n, kind=out_dt) if case["residual"] else None
        if own:
            s["out"] = torch.empty((m, -(-n // 8) * 8), dtype=out_dt, device=dev)[:, :n]
        return s

    q, kv = _lengths(case)
    rows, h, g, d, page = sum(q), case["heads"], case["kv_heads"], case["dim"], case["page"]
    s["q"] = normal(rows, h, d, scale=2.0)  # scores with a deviation of 2 after the scaling by 1/sqrt(dim)
    s["k_new"], s["v_new"] = normal(rows, g, d), normal(rows, g, d)
    s["q_len"], s["q_start"] = ints(q), ints([sum(q[:i]) for i in range(len(q))])
    s["kv_len"] = ints(kv)
    s["max_q"], s["max_kv"] = max(q), max(kv)
    # the pages that a token sees or is written to; the others were given back
    held = []
    for n, t in zip(q, kv):
        first = t - n if case["op"] == "append" else max(0, t - n - case["window"] + 1)
        sunk = 0 if case["op"] == "append" else min(case["sinks"], t)
        held.append(sorted(set(range(first // page, -(-t // page))) | set(range(-(-sunk // page)))))
    pool = sum(map(len, held)) + 3
    perm = torch.randperm(pool, generator=torch.Generator().manual_seed(int(seed))).tolist()
    table = torch.full((len(kv), max(-(-t // page) for t in kv)), -1, dtype=torch.int32)
    at = 0
    for i, which in enumerate(held):
        table[i, which] = torch.tensor(perm[at:at + len(which)], dtype=torch.int32)
        at += len(which)
    s["table"] = table.to(dev)
    s["k_pages"], s["v_pages"] = normal(pool, page, g, d), normal(pool, page, g, d)
    if case["op"] == "append":
        i = torch.arange(case["rot"] // 2, dtype=torch.float64)
        s["inv_freq"] = (10000.0 ** (-2 * i / max(case["rot"], 1))).float().to(dev) if case["rot"] else None
    if own:
        ctx = _context(dev.index)
        s["out"] = torch.empty_like(s["q"])
        kw = dict(q_start=s["q_start"], q_len=s["q_len"], max_q=s["max_q"], max_kv=s["max_kv"])
        if case["op"] == "window":
            s["args"] = ctx.window_args(s["q"], s["k_pages"], s["v_pages"], s["table"], s["kv_len"], s["out"],
                                        window=case["window"], sinks=case["sinks"], k_new=s["k_new"], v_new=s["v_new"],
                                        **kw)
        else:
            s["args"] = ctx.append_args(s["k_new"], s["v_new"], s["k_pages"], s["v_pages"], s["table"], s["kv_len"],
                                        q=s["q"], q_out=s["out"], inv_freq=s["inv_freq"], pairs=case["pairs"], **kw)
    return s


# ---- one pass ------------------------------------------------------------------------------------------------


def run(s):
    op = s["case"]["op"]
    if own:
        if op == "window":
            _context(s["device"]).window(s["args"])
            return {"out": s["out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if op == "append":
            _context(s["device"]).append(s["args"])
            return {"q": s["out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if op == "logprobs":
            _library().logprobs(s["logits"], s["target"], top_n=s["case"]["top"], **s["out"])
            o = s["out"]
            return dict({"logp": o["out_logp"], "entropy": o["out_entropy"]},
                        **({"top_tok": o["out_top_tok"], "top_logp": o["out_top_logp"]} if s["case"]["top"] else {}))
        _library().linear16(s["x"], s["w"], bias=s["bias"], residual=s["residual"], act=s["case"]["act"], out=s["out"])
        return {"out": s["out"]}
    return {"window": _window, "append": _append, "logprobs": _logprobs, "linear": _linear}[op](s)


def _groups(n, size):
    step = max(1, min(n, _GROUP // max(1, size)))
    return [range(i, min(n, i + step)) for i in range(0, n, step)]


def _padded(start, length, most):
    """Numbers of the rows [start, start + length) of each sequence as [B, most], and which of them are there."""
    at = torch.arange(most, device=start.device)
    there = at[None, :] < length[:, None]
    return there, torch.where(there, start[:, None].long() + at, torch.zeros_like(at))


def _place(s, at):
    """Page and slot of positions [B, n] of the sequences (negative page: not there)."""
    page, table = s["case"]["page"], s["table"]
    entry = (at // page).clamp(0, table.shape[1] - 1).long()
    return table.gather(1, entry).long(), (at % page).long()


def _window(s):
    c = s["case"]
    q, kp, vp = s["q"], s["k_pages"], s["v_pages"]
    h, g, d, w, sinks, Q = c["heads"], c["kv_heads"], c["dim"], c["window"], c["sinks"], s["max_q"]
    kl, ql = s["kv_len"].long(), s["q_len"].long()
    there, rows = _padded(s["q_start"], ql, Q)
    at = torch.where(there, (kl - ql)[:, None] + torch.arange(Q, device=q.device), 0)
    pg, slot = _place(s, at)
    kp[pg[there], slot[there]] = s["k_new"][rows[there]]
    vp[pg[there], slot[there]] = s["v_new"][rows[there]]
    out = torch.empty_like(q)
    L = min(s["max_kv"], sinks + w + Q - 1)
    i = torch.arange(L, device=q.device)
    for grp in _groups(c["n_seq"], L * max(g * d, h * Q)):
        sl = slice(grp.start, grp.stop)
        B = len(grp)
        # the keys that some token of the chunk sees: the first ones, then from the first token's window on
        skip = ((kl - ql)[sl] - w + 1 - sinks).clamp(min=0)[:, None]
        key = torch.where(i < sinks, i, i + skip)
        alive = key < kl[sl, None]
        pages, slots = _place(dict(s, table=s["table"][sl]), torch.where(alive, key, 0))
        pages = torch.where(alive, pages, 0)
        k, v = kp[pages, slots].float(), vp[pages, slots].float().masked_fill(~alive[:, :, None, None], 0)
        t = at[sl][:, :, None]
        seen = alive[:, None, :] & (key[:, None, :] <= t) & ((key[:, None, :] > t - w) | (key[:, None, :] < sinks))
        qq = q[rows[sl]].float().view(B, Q, g, h // g, d).permute(0, 2, 3, 1, 4).reshape(B, g, h // g * Q, d)
        sc = torch.matmul(qq, k.permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(d)).view(B, g, h // g, Q, L)
        sc.masked_fill_(~seen[:, None, None], float("-inf"))
        top = sc.amax(-1, keepdim=True)
        top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
        e = sc.sub_(top).exp_()
        total = e.sum(-1, keepdim=True)
        o = torch.matmul(e.view(B, g, h // g * Q, L), v.permute(0, 2, 1, 3)).view(B, g, h // g, Q, d)
        o = (o / torch.where(total == 0, torch.ones_like(total), total)).permute(0, 3, 1, 2, 4).reshape(B, Q, h, d)
        out[rows[sl][there[sl]]] = o[there[sl]].to(out.dtype)
    return {"out": out, "k_pages": kp, "v_pages": vp}


def _turn(x, angle, pairs):
    """x [rows, heads, dim] with its first 2 * angles values turned by angle [rows, angles], in 32 bits."""
    n = angle.shape[1]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    y = x.float().clone()
    a, b = (slice(0, n), slice(n, 2 * n)) if pairs == "halves" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    u, v = x[:, :, a].float(), x[:, :, b].float()
    y[:, :, a], y[:, :, b] = u * cos - v * sin, v * cos + u * sin
    return y.to(x.dtype)


def _append(s):
    c = s["case"]
    kp, vp, Q = s["k_pages"], s["v_pages"], s["max_q"]
    kl, ql = s["kv_len"].long(), s["q_len"].long()
    there, rows = _padded(s["q_start"], ql, Q)
    at = torch.where(there, (kl - ql)[:, None] + torch.arange(Q, device=kp.device), 0)
    pg, slot = _place(s, at)
    pg, slot, rows, at = pg[there], slot[there], rows[there], at[there]
    q, k = s["q"], s["k_new"]
    if c["rot"]:
        pos = torch.zeros(q.shape[0], dtype=torch.float64, device=q.device)
        pos[rows] = at.double()
        angle = pos[:, None] * s["inv_freq"].double()
        q, k = _turn(q, angle, c["pairs"]), _turn(k, angle, c["pairs"])
    else:
        q = q.clone()
    kp[pg, slot], vp[pg, slot] = k[rows], s["v_new"][rows]
    return {"q": q, "k_pages": kp, "v_pages": vp}


def _logprobs(s):
    rows, vocab = s["logits"].shape
    top = s["case"]["top"]
    logp, entropy, tok, lp = [], [], [], []
    for grp in _groups(rows, vocab * 4):
        sl = slice(grp.start, grp.stop)
        x = s["logits"][sl].float()
        t = s["target"][sl].long()[:, None]
        real = t >= 0
        y = x - x.amax(1, keepdim=True)
        e = y.exp()
        total = e.sum(1, keepdim=True, dtype=torch.float64)
        log_z = total.log()
        weighed = (e * y).sum(1, keepdim=True, dtype=torch.float64)
        logp.append(torch.where(real, y.gather(1, t.clamp(min=0)) - log_z, 0.0)[:, 0].float())
        entropy.append(torch.where(real, log_z - weighed / total, 0.0)[:, 0].float())
        if top:
            # by falling logit, then rising index: one whole number for both
            b = (x + 0.0).view(torch.int32).long()
            order = torch.where(b < 0, -(b + 2 ** 31) - 1, b) * 2 ** 20 + (2 ** 20 - 1 - torch.arange(vocab, device=x.device))
            i = order.topk(top, dim=1)[1]
            tok.append(torch.where(real, i, -1).to(torch.int32))
            lp.append(torch.where(real, y.gather(1, i) - log_z, float("-inf")).float())
    out = {"logp": torch.cat(logp), "entropy": torch.cat(entropy)}
    return dict(out, top_tok=torch.cat(tok), top_logp=torch.cat(lp)) if top else out


def _act(y, act):
    if act == "relu":
        return y.clamp(min=0)
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y / math.sqrt(2)))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y / (1 + torch.exp(-y)) if act == "silu" else y


def _linear(s):
    y = s["x"].float() @ s["w"].float().T
    if s["bias"] is not None:
        y += s["bias"].float()
    y = _act(y, s["case"]["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"out": y if s["case"]["wide"] else y.to(s["x"].dtype)}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------


def exact(case, seed):
    plain = own
    globals()["own"] = False  # the inputs alone
    try:
        s = prepare(case, seed)
    finally:
        globals()["own"] = plain
    return {"window": _exact_window, "append": _exact_append, "logprobs": _exact_logprobs, "linear": _exact_linear}[case["op"]](s)


def _exact_window(s):
    c = s["case"]
    h, g, d, w, sinks = c["heads"], c["kv_heads"], c["dim"], c["window"], c["sinks"]
    out = torch.empty_like(s["q"], dtype=torch.float64)
    row = 0
    for i, (n, t) in enumerate(zip(*_lengths(c))):
        first = max(0, t - n - w + 1)
        at = torch.tensor(sorted(set(range(min(sinks, t))) | set(range(first, t))), device=out.device)
        pages, slots = s["table"][i, at // c["page"]].long(), at % c["page"]
        k, v = s["k_pages"][pages, slots], s["v_pages"][pages, slots]
        k[-n:], v[-n:] = s["k_new"][row:row + n], s["v_new"][row:row + n]
        pos = torch.arange(t - n, t, device=out.device)[:, None]
        hidden = (at > pos) | ((at <= pos - w) & (at >= sinks))
        for j in range(h):
            sc = s["q"][row:row + n, j].double() @ k[:, j * g // h].double().T / math.sqrt(d)
            sc[hidden] = -math.inf
            e = torch.exp(sc - sc.max(1, keepdim=True)[0])
            out[row:row + n, j] = (e @ v[:, j * g // h].double()) / e.sum(1, keepdim=True)
        row += n
    return {"out": out, "k_pages": None, "v_pages": None}  # copies, not computed numbers


def _exact_append(s):
    c = s["case"]
    n = c["rot"] // 2
    q, kp, vp = s["q"].double(), s["k_pages"].double(), s["v_pages"].double()
    k = s["k_new"].double()
    row = 0
    for i, (m, t) in enumerate(zip(*_lengths(c))):
        at = torch.arange(t - m, t, device=q.device)
        if n:
            z = torch.polar(torch.ones((m, n), dtype=torch.float64, device=q.device), at[:, None] * s["inv_freq"].double())[:, None]
            for x in (q, k):
                head = x[row:row + m, :, :2 * n]
                # the pairs as complex numbers
                p = head.unflatten(-1, (n, 2)) if c["pairs"] == "neighbours" else head.unflatten(-1, (2, n)).transpose(-1, -2)
                p = torch.view_as_real(torch.view_as_complex(p.contiguous()) * z)
                x[row:row + m, :, :2 * n] = (p if c["pairs"] == "neighbours" else p.transpose(-1, -2)).flatten(-2)
        pages = s["table"][i, at // c["page"]].long()
        kp[pages, at % c["page"]] = k[row:row + m]
        row += m
    return {"q": q, "k_pages": kp, "v_pages": None}


def _exact_logprobs(s):
    rows, top = s["logits"].shape[0], s["case"]["top"]
    if rows * s["logits"].shape[1] > 2 ** 29:
        return None
    logp, entropy, tok, lp = [], [], [], []
    for r in range(rows):
        t = int(s["target"][r])
        if t < 0:
            logp.append(0.0), entropy.append(0.0), tok.append([-1] * top), lp.append([-math.inf] * top)
            continue
        x = s["logits"][r].double()
        z = torch.logsumexp(x, 0)
        p = x - z
        logp.append(float(p[t]))
        entropy.append(float(-(p.exp() * p).sum()))
        if top:
            i = torch.sort(x, descending=True, stable=True)[1][:top]
            tok.append(i.tolist()), lp.append(p[i].tolist())
    out = {"logp": torch.tensor(logp, dtype=torch.float64), "entropy": torch.tensor(entropy, dtype=torch.float64)}
    return dict(out, top_tok=torch.tensor(tok, dtype=torch.int32), top_logp=torch.tensor(lp, dtype=torch.float64)) if top else out


def _exact_linear(s):
    out = []
    for i in range(0, s["x"].shape[0], 1024):
        y = torch.zeros((min(1024, s["x"].shape[0] - i), s["w"].shape[0]), dtype=torch.float64, device=s["x"].device)
        if s["bias"] is not None:
            y += s["bias"].double()
        y = torch.addmm(y, s["x"][i:i + 1024].double(), s["w"].double().T)
        act = s["case"]["act"]
        if act == "relu":
            y = torch.where(y > 0, y, 0.0)
        elif act == "gelu":
            y = y * torch.special.ndtr(y)
        elif act == "gelu_tanh":
            y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
        elif act == "silu":
            y = y * torch.sigmoid(y)
        out.append(y if s["residual"] is None else y + s["residual"][i:i + 1024].double())
    return {"out": torch.cat(out)}
