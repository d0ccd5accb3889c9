"""Measured cases of the paged prompt-and-serving operators: the append of a
chunk of new tokens to a paged cache (per-head norms, rotation and the write in
one pass), the attention of those tokens over the cache, and the scoring of
logits (log probability of given tokens, entropy, rank, top alternatives).

A case is a dict of plain values; prepare() makes its inputs from a seed, run()
makes one pass (the plain form in elementary torch operations, or with
`own = True` the library's calls), work() counts what a pass cannot do without
and exact() computes the same results in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROPE_THETA = 500000.0
EPS = 1e-5


# ------------------------------------------------------------------ the cases
def _append(name, n_seq, chunk, ctx, heads, kv_heads, dim, src, dtype, page, norm, half, layout="head"):
    return {"name": name, "op": "append", "n_seq": n_seq, "chunk": chunk, "ctx": ctx, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "src": src, "dtype": dtype, "page": page, "norm": norm, "half": half,
            "layout": layout}


def _attend(name, n_seq, chunk, ctx, heads, kv_heads, dim, dtype, page, causal=True, softcap=0.0, mixed=False,
            layout="head"):
    return {"name": name, "op": "attend", "n_seq": n_seq, "chunk": chunk, "ctx": ctx, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "page": page, "causal": causal, "softcap": softcap,
            "mixed": mixed, "layout": layout}


def _score(name, rows, vocab, dtype, top, masked):
    return {"name": name, "op": "score", "rows": rows, "vocab": vocab, "dtype": dtype, "top": top, "masked": masked}


def listed():
    return [
        # One decoded token of the 8B shape (32 query, 8 kv heads of 128): the
        # fp32 q|k|v row of the mat-vec goes to the cache; launch latency only.
        _append("append 1 token 8B", 1, 1, 4096, 32, 8, 128, "f32", "f16", 16, False, False),
        # Chunks of four prompts of the 8B shape with normalised heads and the
        # rotation of halves, as a 16-bit matrix product leaves them.
        _append("append 4 chunks 8B bf16", 4, 1031, 4096, 32, 8, 128, "bf16", "bf16", 64, True, True, "token"),
        # A whole prompt of the 70B shape (64 / 8 heads) from fp32 rows.
        _append("append prompt 70B", 1, 8192, 8192, 64, 8, 128, "f32", "f16", 64, True, False),
        # One decoded token at the 8B decode context: latency and the split over keys.
        _attend("decode 1 x 4096 8B", 1, 1, 4096, 32, 8, 128, "f16", 16),
        # A serving batch of the 70B shape, ragged contexts up to its 8192.
        _attend("decode 64 x 8192 70B", 64, 1, 8192, 64, 8, 128, "bf16", 64),
        # A tensor-parallel rank's slice (8 query heads on 1 kv head) at a long context.
        _attend("decode 3 x 32768 slice", 3, 1, 32768, 8, 1, 128, "f16", 128),
        # A chunk of a long prompt: few query tiles, many keys.
        _attend("chunk 512 of 8192 8B", 1, 512, 8192, 32, 8, 128, "f16", 64),
        # A whole prompt of the 8B shape: the matrix products bound it.
        _attend("prompt 8192 8B", 1, 8192, 8192, 32, 8, 128, "bf16", 128),
        # Chunks and single tokens in one batch, odd lengths, heads of 64, capped
        # scores, tokens before heads in a page.
        _attend("mixed batch d64 softcap", 13, 777, 3001, 12, 4, 64, "f16", 24, True, 30.0, True, "token"),
        # The alternatives of one sampled token (the 8B vocabulary).
        _score("score 1 row", 1, 128256, "f32", 20, 0.0),
        # A scored prompt: every row of a 2048-token prompt, 16-bit logits (many ties).
        _score("score 2048 rows bf16", 2048, 128256, "bf16", 8, 0.0),
        # A batch behind a grammar mask (most logits -inf), an odd vocabulary.
        _score("score 333 rows masked", 333, 32003, "f32", 32, 0.9),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    op = rng.choice(["append", "attend", "attend", "score"])
    if op == "score":
        return _score("", _log_int(rng, 1, 2048), _log_int(rng, 97, 160001), rng.choice(["f32", "f16", "bf16"]),
                      rng.choice([0, 1, 5, 8, 20, 32]), rng.choice([0.0, 0.0, 0.5, 0.99]))
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 6, 7, 8])
    dim, dtype = rng.choice([64, 128]), rng.choice(["f16", "bf16"])
    page = rng.choice([1, 8, 16, 16, 24, 32, 33, 64, 64, 128, 256])
    layout = rng.choice(["head", "token"])
    n_seq = _log_int(rng, 1, 64)
    if op == "append":
        chunk = _log_int(rng, 1, 8192)
        ctx = chunk + rng.choice([0, _log_int(rng, 1, 8192)])
        return _append("", n_seq, chunk, ctx, heads, kv_heads, dim, rng.choice(["f32", "f16", "bf16"]), dtype, page,
                       rng.random() < 0.5, rng.random() < 0.5, layout)
    chunk = 1 if rng.random() < 0.4 else _log_int(rng, 2, 4096)
    ctx = chunk + rng.choice([0, _log_int(rng, 1, 32768), _log_int(rng, 1, 32768)])
    return _attend("", n_seq, chunk, ctx, heads, kv_heads, dim, dtype, page, rng.random() < 0.8,
                   rng.choice([0.0, 0.0, 30.0]), rng.random() < 0.3, layout)


def draw(rng):
    most = {op: {"bytes": 0.0, "flops": 0.0} for op in ("append", "attend", "score")}
    for c in listed():
        w = work(c)
        most[c["op"]] = {k: max(most[c["op"]][k], w[k]) for k in w}
    while True:
        c = _draw(rng)
        c.pop("name")
        w = work(c)
        if any(w[k] > most[c["op"]][k] for k in w):
            continue
        if c["op"] == "attend":   # the plain form's padded scores stay within those of the largest listed case
            q, kv = _lengths(c)
            if len(q) * max(q) * max(kv) * c["heads"] > 8192 * 8192 * 32 or len(q) * max(kv) * c["kv_heads"] > 1 << 23:
                continue
        return c


def _lengths(case):
    """(new tokens, total tokens) of each sequence: a function of the case alone."""
    r = random.Random("%(n_seq)d %(chunk)d %(ctx)d %(heads)d %(page)d" % case)
    n, chunk, ctx = case["n_seq"], case["chunk"], case["ctx"]
    q = [chunk] + [r.randint(max(1, chunk // 8), chunk) for _ in range(n - 1)]
    if case.get("mixed"):   # every other sequence decodes one token
        q = [1 if i % 2 else v for i, v in enumerate(q)]
    kv = [ctx] + [r.randint(max(v, ctx // 8), max(v, ctx)) for v in q[1:]]
    return q, kv


def work(case):
    if case["op"] == "score":
        size = DTYPES[case["dtype"]].itemsize
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        return {"bytes": float(rows * (vocab * size + 4 + 12 + 8 * top)), "flops": 5.0 * rows * vocab}
    q, kv = _lengths(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        size = DTYPES[case["src"]].itemsize
        values = sum(q) * (heads + 2 * kv_heads) * dim
        return {"bytes": float(values * (size + 2) + sum(q) * dim * 4), "flops": 8.0 * values}
    pairs = sum((n * t - n * (n - 1) // 2) if case["causal"] else n * t for n, t in zip(q, kv))
    cache = sum(kv) * kv_heads * dim * 2 * 2
    rows = sum(q) * heads
    return {"bytes": float(cache + rows * (dim * 2 * 2 + 4)), "flops": 4.0 * dim * heads * pairs}


# ------------------------------------------------------------------ the inputs
def _rope_table(n, dim):
    """[n, dim/2, 2] of (cos, sin), the angles in 64 bits."""
    pos = torch.arange(n, dtype=torch.float64, device="cuda")[:, None]
    inv = ROPE_THETA ** (-2.0 * torch.arange(dim // 2, dtype=torch.float64, device="cuda") / dim)
    return torch.stack([(pos * inv).cos(), (pos * inv).sin()], dim=-1).float().contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    host = np.random.RandomState(seed % (1 << 31))
    if case["op"] == "score":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn(rows, vocab, generator=g, device="cuda") * 3.0
        if case["masked"]:   # the given token and some others stay allowed
            x.masked_fill_(torch.rand(rows, vocab, generator=g, device="cuda") < case["masked"], -math.inf)
        tokens = torch.from_numpy(host.randint(0, vocab, rows).astype(np.int32)).cuda()
        x[torch.arange(rows, device="cuda"), tokens.long()] = torch.randn(rows, generator=g, device="cuda") + 4.0
        return {"case": case, "logits": x.to(DTYPES[case["dtype"]]), "tokens": tokens}
    q, kv = _lengths(case)
    n, page, dtype = case["n_seq"], case["page"], DTYPES[case["dtype"]]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    pages = [-(-t // page) for t in kv]
    n_pages = sum(pages) + 3
    order = host.permutation(n_pages).astype(np.int32)
    table = np.full((n, max(pages)), -1, np.int32)   # entries past a sequence's pages are never read
    at = 0
    for i, p in enumerate(pages):
        table[i, :p] = order[at:at + p]
        at += p
    q_start = np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
    shape = (n_pages, kv_heads, page, dim) if case["layout"] == "head" else (n_pages, page, kv_heads, dim)
    s = {"case": case, "table": torch.from_numpy(table).cuda(), "q_start": torch.from_numpy(q_start).cuda(),
         "kv_len": torch.tensor(kv, dtype=torch.int32, device="cuda"), "n_pages": n_pages, "max_q": max(q),
         "max_kv": max(kv), "n_tokens": int(q_start[-1])}
    if case["op"] == "append":
        width = (heads + 2 * kv_heads) * dim
        s["qkv"] = (torch.randn(s["n_tokens"], width, generator=g, device="cuda") * 1.5).to(DTYPES[case["src"]])
        s["k"] = torch.zeros(shape, dtype=dtype, device="cuda")
        s["v"] = torch.zeros(shape, dtype=dtype, device="cuda")
        s["rope"] = _rope_table(max(kv), dim)
        s["q_norm"] = torch.rand(dim, generator=g, device="cuda") * 0.2 + 0.9 if case["norm"] else None
        s["k_norm"] = torch.rand(dim, generator=g, device="cuda") * 0.2 + 0.9 if case["norm"] else None
    else:
        s["q"] = (torch.randn(s["n_tokens"], heads, dim, generator=g, device="cuda") * 1.5).to(dtype)
        s["k"] = torch.randn(shape, generator=g, device="cuda", dtype=dtype)
        s["v"] = torch.randn(shape, generator=g, device="cuda", dtype=dtype)
    return s


# ------------------------------------------------------------------ the plain forms
def _where(s):
    """Of each new token: its sequence, its index among the sequence's new tokens, its position."""
    t = torch.arange(s["n_tokens"], device="cuda")
    start = s["q_start"].long()
    seq = torch.searchsorted(start, t, right=True) - 1
    i = t - start[seq]
    return seq, i, s["kv_len"].long()[seq] - (start[seq + 1] - start[seq]) + i


def _normed(x, w):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _rotated(x, cs, half):
    c, d = cs[:, None, :, 0], cs[:, None, :, 1]
    h = x.shape[-1] // 2
    a, b = (x[..., :h], x[..., h:]) if half else (x[..., 0::2], x[..., 1::2])
    y = (a * c - b * d, a * d + b * c)
    return torch.cat(y, -1) if half else torch.stack(y, -1).flatten(-2)


def _plain_append(s):
    c = s["case"]
    heads, kv_heads, dim = c["heads"], c["kv_heads"], c["dim"]
    x = s["qkv"].float().view(-1, heads + 2 * kv_heads, dim)
    seq, _, pos = _where(s)
    cs = s["rope"][pos]
    q = _rotated(_normed(x[:, :heads], s["q_norm"]), cs, c["half"]).to(s["k"].dtype)
    k = _rotated(_normed(x[:, heads:heads + kv_heads], s["k_norm"]), cs, c["half"])
    page, off = s["table"][seq, pos // c["page"]].long(), pos % c["page"]
    at = (page[:, None], torch.arange(kv_heads, device="cuda")[None], off[:, None])
    if c["layout"] == "token":
        at = (at[0], at[2], at[1])
    s["k"][at] = k.to(s["k"].dtype)
    s["v"][at] = x[:, heads + kv_heads:].to(s["v"].dtype)
    return {"q": q, "k": s["k"], "v": s["v"]}


def _plain_attend(s):
    c = s["case"]
    heads, kv_heads, dim, n = c["heads"], c["kv_heads"], c["dim"], c["n_seq"]
    group = heads // kv_heads
    seq, i, _ = _where(s)

    def rows(pages):   # [n_seq, kv_heads, max_kv, dim] in 32 bits
        x = pages[s["table"].long().clamp(min=0)]
        x = x.permute(0, 2, 1, 3, 4) if c["layout"] == "head" else x.permute(0, 3, 1, 2, 4)
        return x.reshape(n, kv_heads, -1, dim)[:, :, :s["max_kv"]].float()

    q = torch.zeros(n, s["max_q"], heads, dim, device="cuda")
    q[seq, i] = s["q"].float()
    q = q.view(n, s["max_q"], kv_heads, group, dim).permute(0, 2, 1, 3, 4).reshape(n, kv_heads, -1, dim)
    x = q @ rows(s["k"]).transpose(-1, -2)
    x *= 1.0 / math.sqrt(dim)
    if c["softcap"]:
        x = x.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    new = s["q_start"].long().diff()
    key = torch.arange(s["max_kv"], device="cuda")
    row = torch.arange(s["max_q"], device="cuda")
    last = s["kv_len"].long()[:, None].expand(n, s["max_q"])
    if c["causal"]:
        last = last - new[:, None] + row + 1
        last = torch.minimum(last, s["kv_len"].long()[:, None])
    seen = (key < last[:, :, None])[:, None, :, None].expand(n, 1, s["max_q"], group, s["max_kv"])
    x = x.view(n, kv_heads, s["max_q"], group, s["max_kv"]).masked_fill_(~seen, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = x.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = p.view(n, kv_heads, -1, s["max_kv"]) @ rows(s["v"])
    o = o.view(n, kv_heads, s["max_q"], group, dim) / total
    lse = (m + total.log())[..., 0]
    o = o.permute(0, 2, 1, 3, 4).reshape(n, s["max_q"], heads, dim)[seq, i]
    lse = lse.permute(0, 2, 1, 3).reshape(n, s["max_q"], heads)[seq, i]
    return {"o": o.to(s["q"].dtype), "lse": lse}


def _plain_score(s):
    c = s["case"]
    x, tok = s["logits"].float(), s["tokens"].long()[:, None]
    given = x.gather(1, tok)
    index = torch.arange(c["vocab"], device="cuda")
    rank = ((x > given) | ((x == given) & (index < tok))).sum(1).int()
    value, at = torch.sort(x, dim=1, descending=True, stable=True)
    value, at = value[:, :c["top"]], at[:, :c["top"]].int()
    m = x.amax(1, keepdim=True)
    x = x - m
    e = x.exp()
    total = e.sum(1, keepdim=True)
    log_total = total.log()
    entropy = (log_total - (e * x.clamp(min=-1e30)).sum(1, keepdim=True) / total)[:, 0]
    top = value - m - log_total
    at = torch.where(value == -math.inf, torch.full_like(at, -1), at)
    return {"logprob": (given - m - log_total)[:, 0], "entropy": entropy, "rank": rank, "top_index": at,
            "top_logprob": top}


# ------------------------------------------------------------------ the library's calls
def _own(s):
    import p100_b200 as P
    c = s["case"]
    if c["op"] == "score":
        if "ws" not in s:
            s["ws"] = P.logprobs_workspace(c["rows"], c["vocab"], c["top"])
        r = P.logprobs(s["logits"], s["tokens"], top_k=c["top"], ws=s["ws"])
        return {"logprob": r.logprob, "entropy": r.entropy, "rank": r.rank, "top_index": r.top_index,
                "top_logprob": r.top_logprob}
    if "desc" not in s:
        dim, page, kv_heads = c["dim"], c["page"], c["kv_heads"]
        tokens_first = c["layout"] == "token"
        s["desc"] = P.PagedDesc(
            n_seq=c["n_seq"], n_tokens=s["n_tokens"], max_q=s["max_q"], n_head_q=c["heads"], n_head_kv=kv_heads,
            head_dim=dim, dtype=P.BF16 if c["dtype"] == "bf16" else P.F16, page_size=page, n_pages=s["n_pages"],
            max_pages=s["table"].shape[1], softcap=c.get("softcap", 0.0), causal=c.get("causal", True),
            head_stride=dim if tokens_first else 0, token_stride=kv_heads * dim if tokens_first else 0)
    if c["op"] == "append":
        q = P.paged_append(s["desc"], s["qkv"], s["table"], s["q_start"], s["kv_len"], s["k"], s["v"],
                           rope_cs=s["rope"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, rope_half=c["half"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    if "ws" not in s:
        s["ws"] = P.fa_paged_workspace(s["desc"])
    o, lse = P.fa_paged(s["desc"], s["q"], s["k"], s["v"], s["table"], s["q_start"], s["kv_len"], ws=s["ws"])
    return {"o": o, "lse": lse}


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "attend": _plain_attend, "score": _plain_score}[state["case"]["op"]](state)


# ------------------------------------------------------------------ 64 bits
def _exact_score(s):
    c = s["case"]
    out = {k: [] for k in ("logprob", "entropy", "top_logprob")}
    for x, t in zip(s["logits"], s["tokens"].tolist()):
        y = torch.log_softmax(x.double(), 0)
        p = y.exp()
        out["logprob"].append(y[t])
        out["entropy"].append(-torch.where(p > 0, p * y, torch.zeros_like(y)).sum())
        out["top_logprob"].append(torch.topk(y, c["top"]).values)
    out = {k: torch.stack(v) for k, v in out.items()}
    return {**out, "rank": None, "top_index": None}


def _exact_append(s):
    c = s["case"]
    heads, kv_heads, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    q_start, kv_len = s["q_start"].tolist(), s["kv_len"].tolist()
    k_out, v_out = s["k"].double(), s["v"].double()
    if c["layout"] == "token":
        k_out, v_out = k_out.transpose(1, 2).contiguous(), v_out.transpose(1, 2).contiguous()
    rotated = []
    for b in range(c["n_seq"]):
        x = s["qkv"][q_start[b]:q_start[b + 1]].double().view(-1, heads + 2 * kv_heads, dim)
        n = x.shape[0]
        pos = torch.arange(kv_len[b] - n, kv_len[b], device="cuda")
        turn = torch.view_as_complex(s["rope"][pos].double())[:, None]
        done = []
        for part, w in ((x[:, :heads], s["q_norm"]), (x[:, heads:heads + kv_heads], s["k_norm"])):
            if w is not None:
                part = part / (part.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt() * w.double()
            pairs = part.unflatten(-1, (2, dim // 2)).transpose(-1, -2) if c["half"] else part.unflatten(-1, (dim // 2, 2))
            y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            done.append((y.transpose(-1, -2) if c["half"] else y).flatten(-2))
        rotated.append(done[0])
        slot = s["table"][b].long()[pos // page]
        k_out[slot, :, pos % page] = done[1]
        v_out[slot, :, pos % page] = x[:, heads + kv_heads:]
    if c["layout"] == "token":
        k_out, v_out = k_out.transpose(1, 2).contiguous(), v_out.transpose(1, 2).contiguous()
    return {"q": torch.cat(rotated), "k": k_out, "v": v_out}


def _exact_attend(s):
    c = s["case"]
    heads, kv_heads, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    group = heads // kv_heads
    q_start, kv_len = s["q_start"].tolist(), s["kv_len"].tolist()
    o = torch.zeros(s["n_tokens"], heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["n_tokens"], heads, dtype=torch.float64, device="cuda")
    for b in range(c["n_seq"]):
        t, lo, hi = kv_len[b], q_start[b], q_start[b + 1]
        where = torch.arange(t, device="cuda")
        slot, off = s["table"][b].long()[where // page], where % page
        for h in range(kv_heads):
            k, v = ((x[slot, h, off] if c["layout"] == "head" else x[slot, off, h]).double() for x in (s["k"], s["v"]))
            for g in range(h * group, (h + 1) * group):
                z = torch.mv if hi - lo == 1 else torch.mm
                y = (z(k, s["q"][lo, g].double())[None] if hi - lo == 1 else z(s["q"][lo:hi, g].double(), k.T)) / dim ** 0.5
                if c["softcap"]:
                    y = torch.tanh(y / c["softcap"]) * c["softcap"]
                if c["causal"] and hi - lo > 1:
                    y = torch.where(torch.ones_like(y, dtype=torch.bool).tril(t - (hi - lo)), y, -math.inf)
                lse[lo:hi, g] = torch.logsumexp(y, -1)
                o[lo:hi, g] = torch.softmax(y, -1) @ v
    return {"o": o, "lse": lse}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        if work(case)["flops"] > 1.2e12:
            return None
        return _exact_attend(s)
    return _exact_score(s) if case["op"] == "score" else _exact_append(s)
