"""Measured cases of decoding with trees of drafted tokens over a paged cache:
the plan of a step (block tables, starts and slots from the requests' lengths),
the tree's masks and positions, the append of the drafted tokens with their
rotation at those positions, the attention under the tree's mask, and the move
of the accepted tokens' keys and values to their final rows.

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
EPS = 1e-5
# kinds of scaled rotary frequencies, with the arguments the cases use
SCALING = {
    "none": {},
    "linear": {"factor": 4.0},
    "ntk": {"factor": 8.0},
    "bands": {"factor": 8.0, "low": 1.0, "high": 4.0, "original": 8192},
    "yarn": {"factor": 16.0, "low": 1.0, "high": 32.0, "original": 1024},
    "divisors": {"mscale": 1.19},
}
THETA = 500000.0


# ------------------------------------------------------------------ the cases
def _plan(name, n_seq, draft, ctx, page):
    return {"name": name, "op": "plan", "n_seq": n_seq, "draft": draft, "ctx": ctx, "page": page}


def _mask(name, n_seq, draft, ctx, deep):
    return {"name": name, "op": "mask", "n_seq": n_seq, "draft": draft, "ctx": ctx, "deep": deep}


def _append(name, n_seq, draft, ctx, heads, kv_heads, dim, src, dtype, page, norm, half, rope_dim, scaling, tree,
            layout="head"):
    return {"name": name, "op": "append", "n_seq": n_seq, "draft": draft, "ctx": ctx, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "src": src, "dtype": dtype, "page": page, "norm": norm, "half": half,
            "rope_dim": rope_dim, "scaling": scaling, "tree": tree, "layout": layout}


def _attend(name, n_seq, draft, ctx, heads, kv_heads, dim, dtype, page, softcap=0.0, layout="head"):
    return {"name": name, "op": "attend", "n_seq": n_seq, "draft": draft, "ctx": ctx, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "page": page, "softcap": softcap, "layout": layout}


def _keep(name, n_seq, draft, ctx, kv_heads, dim, dtype, page, layout="head"):
    return {"name": name, "op": "keep", "n_seq": n_seq, "draft": draft, "ctx": ctx, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype, "page": page, "layout": layout}


def listed():
    return [
        # A small serving batch that drafts a few tokens a request; latency only.
        _plan("plan 16 x 4 drafts", 16, 4, 4096, 16),
        # The most requests of one call, drafts of up to 16 tokens, small pages.
        _plan("plan 1024 x 16 drafts", 1024, 16, 8192, 16),
        # One request's tree of 16 tokens.
        _mask("tree of 16", 1, 16, 4096, 6),
        # A batch of large trees, the deep ones nearly chains.
        _mask("64 trees of 250", 64, 250, 8192, 60),
        # One tree of the 8B shape (32 query, 8 kv heads of 128): fp32 rows of
        # the mat-vec, a part of each head rotated; launch latency only.
        _append("append 1 tree 8B half the head", 1, 8, 4096, 32, 8, 128, "f32", "f16", 16, False, False, 64, "none",
                True),
        # Trees of 64 requests as a 16-bit matrix product leaves them, normalised
        # heads, halves, positions in a context scaled sixteenfold.
        _append("append 64 trees 70B yarn", 64, 64, 8192, 64, 8, 128, "bf16", "bf16", 64, True, True, 128, "yarn",
                True, "token"),
        # One request's tree of 16 tokens at the 8B decode context: latency and
        # the split over keys.
        _attend("attend 1 tree of 16 x 4096 8B", 1, 16, 4096, 32, 8, 128, "f16", 16),
        # A serving batch of the 70B shape, trees of up to 8, ragged contexts:
        # the cache's bytes bound it.
        _attend("attend 48 trees of 8 x 8192 70B", 48, 8, 8192, 64, 8, 128, "bf16", 64),
        # Large trees at long contexts: bytes and products are alike.
        _attend("attend 8 trees of 64 x 32768 8B", 8, 64, 32768, 32, 8, 128, "bf16", 128),
        # Short drafts on a few heads of 64, capped scores, odd pages, tokens
        # before heads in a page.
        _attend("attend 13 trees of 5 x 3001 d64", 13, 5, 3001, 12, 4, 64, "f16", 24, 30.0, "token"),
        # The accepted tokens of one 70B layer's pages, and of one request.
        _keep("keep 1 of 8 8B", 1, 8, 4096, 8, 128, "f16", 16),
        _keep("keep 64 of 64 70B", 64, 64, 8192, 8, 128, "bf16", 64, "token"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    op = rng.choice(["plan", "mask", "append", "attend", "attend", "attend", "keep"])
    page = rng.choice([1, 8, 16, 16, 24, 32, 33, 64, 64, 128, 256])
    n_seq = _log_int(rng, 1, 64)
    if op == "plan":
        return _plan("", _log_int(rng, 1, 1024), _log_int(rng, 1, 64), _log_int(rng, 64, 8192), max(8, page))
    if op == "mask":
        draft = _log_int(rng, 1, 500)
        return _mask("", n_seq, draft, draft + _log_int(rng, 1, 8192), _log_int(rng, 1, 64))
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 6, 7, 8])
    dim, dtype = rng.choice([64, 128]), rng.choice(["f16", "bf16"])
    layout = rng.choice(["head", "token"])
    if op == "append":
        tree = rng.random() < 0.7
        draft = _log_int(rng, 1, 64 if tree else 4096)
        rope_dim = rng.choice([dim, dim, dim // 2, dim // 4, 3 * dim // 4, 20, 40])
        return _append("", n_seq, draft, draft + _log_int(rng, 1, 16384), heads, kv_heads, dim,
                       rng.choice(["f32", "f16", "bf16"]), dtype, page, rng.random() < 0.5, rng.random() < 0.5, rope_dim,
                       rng.choice(list(SCALING)), tree, layout)
    draft = _log_int(rng, 1, 100)
    ctx = draft + rng.choice([0, _log_int(rng, 1, 32768), _log_int(rng, 1, 32768)])
    if op == "keep":
        return _keep("", n_seq, draft, ctx, kv_heads, dim, dtype, page, layout)
    return _attend("", n_seq, draft, ctx, heads, kv_heads, dim, dtype, page, rng.choice([0.0, 0.0, 30.0]), layout)


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        most[c["op"]] = {k: max(most.get(c["op"], w)[k], w[k]) for k in w}
    while True:
        c = _draw(rng)
        c.pop("name")
        w = work(c)
        if any(w[k] > most[c["op"]][k] for k in w):
            continue
        if c["op"] in ("attend", "append", "keep"):   # what the plain form and the pages hold stays within the largest listed case
            q, kv = _lengths(c)
            if c["op"] == "attend" and len(q) * max(q) * max(kv) * c["heads"] > 8 * 64 * 32768 * 32:
                continue
            if len(q) * max(kv) * c["kv_heads"] > 64 * 65536:
                continue
        return c


def _lengths(case):
    """(new tokens, total tokens) of each sequence: a function of the case alone."""
    r = random.Random("%(op)s %(n_seq)d %(draft)d %(ctx)d" % case)
    n, draft, ctx = case["n_seq"], case["draft"], case["ctx"]
    q = [draft] + [r.randint(max(1, draft // 4), draft) for _ in range(n - 1)]
    return q, [ctx] + [r.randint(max(v, ctx // 8), max(v, ctx)) for v in q[1:]]


def work(case):
    q, kv = _lengths(case)
    n, tokens = len(q), sum(q)
    if case["op"] == "plan":   # the drafts of the last step given back, new ones taken
        page = case["page"]
        pages = sum(-(-t // page) - -(-(t - m) // page) for m, t in zip(q, kv))
        rows = n * case["draft"]
        return {"bytes": float(2 * 24 * n + 2 * 12 * rows + 2 * 8 * pages), "flops": float(2 * rows + n)}
    if case["op"] == "mask":
        words = -(-case["draft"] // 32)
        return {"bytes": float(tokens * (4 + 4 + 4 * words) + 8 * n), "flops": float(tokens)}
    kv_heads, dim = case["kv_heads"], case["dim"]
    if case["op"] == "keep":
        kept = sum(_kept(m) for m in q)
        return {"bytes": float(kept * kv_heads * dim * 2 * 2 * 2 + 4 * kept), "flops": 0.0}
    heads = case["heads"]
    if case["op"] == "append":
        size = DTYPES[case["src"]].itemsize
        values = tokens * (heads + 2 * kv_heads) * dim
        return {"bytes": float(values * (size + 2) + tokens * 4), "flops": 8.0 * values}
    rows = tokens * heads
    pairs = sum(m * (t - m + 1) for m, t in zip(q, kv))
    return {"bytes": float(sum(kv) * kv_heads * dim * 2 * 2 + rows * (dim * 2 * 2 + 4)), "flops": 4.0 * dim * heads * pairs}


def _kept(n):
    """Accepted tokens of a tree of n: about half of a path of log length, as many for every seed."""
    return min(n, 1 + n.bit_length() // 2 + n // 24)


# ------------------------------------------------------------------ the inputs
def _trees(host, q, deep):
    """Parents of every sequence's drafted tokens: earlier ones of the tree, -1 behind the context."""
    out = []
    for n in q:
        depth, parent = [], []
        for i in range(n):
            p = -1 if i == 0 or host.rand() < 1.5 / n else int(host.randint(max(0, i - 1 - n // 4), i))
            while p >= 0 and depth[p] + 1 >= deep:
                p = parent[p]
            parent.append(p)
            depth.append(0 if p < 0 else depth[p] + 1)
        out += parent
    return np.array(out, np.int32)


def _masks(q, parent, words):
    """Bit j of a token's row: it sees token j of its own tree (its ancestors and itself)."""
    out = np.zeros((len(parent), words), np.uint32)
    at = 0
    for n in q:
        for i in range(n):
            if parent[at + i] >= 0:
                out[at + i] = out[at + parent[at + i]]
            out[at + i, i // 32] |= np.uint32(1 << (i % 32))
        at += n
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    host = np.random.RandomState(seed % (1 << 31))
    q, kv = _lengths(case)
    n = case["n_seq"]
    q_start = np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
    s = {"case": case, "n_tokens": int(q_start[-1]), "max_q": max(q), "max_kv": max(kv), "words": -(-max(q) // 32),
         "q_start": torch.from_numpy(q_start).cuda(), "kv_len": torch.tensor(kv, dtype=torch.int32, device="cuda")}
    if case["op"] == "mask":
        s["parent"] = torch.from_numpy(_trees(host, q, case["deep"])).cuda()
        return s
    page = case["page"]
    pages = [-(-t // page) for t in kv]
    n_pages = sum(pages) + 3
    order = host.permutation(n_pages).astype(np.int32)
    table = np.full((n, max(pages)), -1, np.int32)
    at = 0
    for i, p in enumerate(pages):
        table[i, :p] = order[at:at + p]
        at += p
    s["table"], s["n_pages"] = torch.from_numpy(table).cuda(), n_pages
    if case["op"] == "plan":   # the state after a step: every draft has its pages
        s["n_tokens"] = n * case["draft"]
        s["length"] = s["kv_len"] - torch.tensor(q, dtype=torch.int32, device="cuda")
        s["n_new"] = torch.tensor(q, dtype=torch.int32, device="cuda")
        s["none"] = torch.zeros_like(s["n_new"])
        s["held"] = torch.tensor(pages, dtype=torch.int32, device="cuda")
        free = np.full(n_pages, -1, np.int32)
        free[:n_pages - at] = order[at:]
        s["pool"] = torch.from_numpy(np.concatenate([[n_pages - at, 0], free]).astype(np.int32)).cuda()
        return s
    kv_heads, dim, dtype = case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    shape = (n_pages, kv_heads, page, dim) if case["layout"] == "head" else (n_pages, page, kv_heads, dim)
    if case["op"] == "append":
        heads = case["heads"]
        width = (heads + 2 * kv_heads) * dim
        s["qkv"] = (torch.randn(s["n_tokens"], width, generator=g, device="cuda") * 1.5).to(DTYPES[case["src"]])
        s["k"] = torch.zeros(shape, dtype=dtype, device="cuda")
        s["v"] = torch.zeros(shape, dtype=dtype, device="cuda")
        s["q_norm"] = torch.rand(dim, generator=g, device="cuda") * 0.2 + 0.9 if case["norm"] else None
        s["k_norm"] = torch.rand(dim, generator=g, device="cuda") * 0.2 + 0.9 if case["norm"] else None
        s["scaling"] = dict(SCALING[case["scaling"]])
        if case["scaling"] == "divisors":
            s["scaling"]["divisors"] = [1.0 + 30.0 * (i / case["rope_dim"]) ** 2 for i in range(case["rope_dim"] // 2)]
        s["position"] = None
        if case["tree"]:
            parent = _trees(host, q, 8)
            depth = np.zeros(len(parent), np.int32)
            base = np.repeat(q_start[:-1], q)
            for i, p in enumerate(parent):
                depth[i] = 0 if p < 0 else depth[base[i] + p] + 1
            s["position"] = torch.from_numpy(np.repeat(np.array(kv) - np.array(q), q).astype(np.int32) + depth).cuda()
        return s
    s["k"] = torch.randn(shape, generator=g, device="cuda", dtype=dtype)
    s["v"] = torch.randn(shape, generator=g, device="cuda", dtype=dtype)
    if case["op"] == "keep":
        keep = np.full(s["n_tokens"], -1, np.int32)
        for i, m in enumerate(q):
            keep[q_start[i]:q_start[i] + _kept(m)] = np.sort(host.permutation(m)[:_kept(m)])
        s["keep"] = torch.from_numpy(keep).cuda()
        s["keep_len"] = torch.tensor([_kept(m) for m in q], dtype=torch.int32, device="cuda")
        return s
    s["q"] = (torch.randn(s["n_tokens"], case["heads"], dim, generator=g, device="cuda") * 1.5).to(dtype)
    s["mask"] = torch.from_numpy(_masks(q, _trees(host, q, 8), s["words"]).view(np.int32)).cuda()
    return s


# ------------------------------------------------------------------ the plain forms
def _where(s):
    """Of each new token: its sequence, its index among the sequence's new tokens."""
    t = torch.arange(s["n_tokens"], device="cuda")
    seq = torch.searchsorted(s["q_start"].long(), t, right=True) - 1
    return seq, t - s["q_start"].long()[seq]


def _slots(s, seq, pos):
    """The page and the row in it of a token."""
    page = s["case"]["page"]
    return s["table"][seq, pos // page].long(), pos % page


def _plain_plan(s, n_new):
    page, n_tokens = s["case"]["page"], s["n_tokens"]
    table, held, pool, length = s["table"], s["held"], s["pool"], s["length"]
    kv_len = length + n_new
    need = (kv_len + page - 1) // page
    col = torch.arange(table.shape[1], device="cuda", dtype=torch.int32)
    give = ((col >= need[:, None]) & (col < held[:, None])).flatten()
    take = ((col >= held[:, None]) & (col < need[:, None])).flatten()
    top = pool[0] + give.sum() - 1
    entries, stack = table.view(-1), pool[2:]
    # returned pages, the first on top; then pages from the top on
    stack[(top - (give.cumsum(0) - 1))[give]] = entries[give]
    entries[give] = -1
    entries[take] = stack[(top - (take.cumsum(0) - 1))[take]]
    pool[0] = top + 1 - take.sum()
    pool[1] = 0
    held.copy_(need)
    q_start = torch.cat([torch.zeros_like(n_new[:1]), n_new.cumsum(0).int()])
    t = torch.arange(n_tokens, device="cuda")
    seq = (torch.searchsorted(q_start.long(), t, right=True) - 1).clamp(max=len(n_new) - 1)
    pos = length.long()[seq] + t - q_start.long()[seq]
    live = t < q_start[-1]
    entry = table[seq, torch.where(live, pos // page, 0)].long()
    slot = torch.where(live, entry * page + pos % page, -1)
    return {"q_start": q_start, "kv_len": kv_len, "slot": slot, "position": torch.where(live, pos, -1).int(),
            "table": table, "held": held, "pool": pool}


def _plain_mask(s):
    seq, i = _where(s)
    n, most, words = s["case"]["n_seq"], s["max_q"], s["words"]
    # hop[t]: an ancestor of node t (`most`: none left), doubled in distance each round
    hop = torch.full((n, most + 1), most, dtype=torch.long, device="cuda")
    hop[seq, i] = torch.where(s["parent"] < 0, most, s["parent"].long())
    sees = torch.eye(most + 1, dtype=torch.bool, device="cuda").expand(n, -1, -1).clone()
    sees[:, most] = False
    for _ in range(max(1, most.bit_length())):
        sees = sees | sees.gather(1, hop[:, :, None].expand(-1, -1, most + 1))
        hop = hop.gather(1, hop)
    sees = sees[seq, i, :most]
    depth = sees.sum(1) - 1
    bits = torch.nn.functional.pad(sees, (0, 32 * words - most)).view(-1, words, 32).long()
    value = (bits << torch.arange(32, device="cuda")).sum(-1)
    ctx = s["kv_len"].long() - s["q_start"].long().diff()
    return {"mask": torch.where(value >= 1 << 31, value - (1 << 32), value).int(), "position": (ctx[seq] + depth).int()}


def _normed(x, w):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _frequencies(c, a):
    """Radians a token of each pair and the factor of the rotated values, in 64 bits."""
    r, kind = c["rope_dim"], c["scaling"]
    i = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    theta = THETA * (a["factor"] ** (r / (r - 2)) if kind == "ntk" else 1.0)
    f = theta ** (-2.0 * i / r)
    if kind == "linear":
        f = f / a["factor"]
    if kind == "bands":
        turns = a["original"] * f / (2 * math.pi)
        f = f * torch.lerp(torch.full_like(f, 1 / a["factor"]), torch.ones_like(f),
                           ((turns - a["low"]) / (a["high"] - a["low"])).clamp(0, 1))
    if kind == "yarn":
        at = [r * math.log(a["original"] / (b * 2 * math.pi)) / (2 * math.log(THETA)) for b in (a["high"], a["low"])]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), r - 1)
        ramp = ((i - lo) / (hi - lo if hi > lo else 0.001)).clamp(0, 1)
        f = f * (ramp / a["factor"] + (1 - ramp))
    if kind == "divisors":
        f = f / torch.tensor(a["divisors"], dtype=torch.float64, device="cuda")
    return f, 0.1 * math.log(a["factor"]) + 1 if kind == "yarn" else a.get("mscale", 1.0)


def _plain_append(s):
    c = s["case"]
    heads, kv_heads, dim, r = c["heads"], c["kv_heads"], c["dim"], c["rope_dim"]
    x = s["qkv"].float().view(-1, heads + 2 * kv_heads, dim)
    seq, i = _where(s)
    pos = s["kv_len"].long()[seq] - s["q_start"].long().diff()[seq] + i
    f, m = _frequencies(c, s["scaling"])
    angle = (pos if s["position"] is None else s["position"]).double()[:, None] * f
    cos, sin = (angle.cos() * m).float()[:, None], (angle.sin() * m).float()[:, None]

    def rotated(y):
        z = y[..., :r]
        a, b = (z[..., :r // 2], z[..., r // 2:]) if c["half"] else (z[..., 0::2], z[..., 1::2])
        t = (a * cos - b * sin, a * sin + b * cos)
        t = torch.cat(t, -1) if c["half"] else torch.stack(t, -1).flatten(-2)
        return torch.cat([t, y[..., r:]], -1)

    q = rotated(_normed(x[:, :heads], s["q_norm"])).to(s["k"].dtype)
    k = rotated(_normed(x[:, heads:heads + kv_heads], s["k_norm"]))
    page, off = _slots(s, seq, pos)
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
    seq, i = _where(s)

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
    # the context is seen by all, the tree's tokens by the bits of the mask
    ctx = s["kv_len"].long() - s["q_start"].long().diff()
    bits = torch.zeros(n, s["max_q"], s["words"] * 32, dtype=torch.bool, device="cuda")
    bits[seq, i] = ((s["mask"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1).bool().flatten(1)
    node = torch.arange(s["max_kv"], device="cuda") - ctx[:, None]
    tree = bits.gather(2, node.clamp(0, s["words"] * 32 - 1)[:, None].expand(n, s["max_q"], -1))
    inside = torch.arange(s["max_kv"], device="cuda") < s["kv_len"].long()[:, None]
    seen = (node < 0)[:, None] | (tree & inside[:, None])
    x = x.view(n, kv_heads, s["max_q"], group, s["max_kv"]).masked_fill_(~seen[:, None, :, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = x.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = p.view(n, kv_heads, -1, s["max_kv"]) @ rows(s["v"])
    o = o.view(n, kv_heads, s["max_q"], group, dim) / total
    lse = (m + total.log())[..., 0]
    o = o.permute(0, 2, 1, 3, 4).reshape(n, s["max_q"], heads, dim)[seq, i]
    lse = lse.permute(0, 2, 1, 3).reshape(n, s["max_q"], heads)[seq, i]
    return {"o": o.to(s["q"].dtype), "lse": lse}


def _plain_keep(s):
    c = s["case"]
    seq, i = _where(s)
    ctx = s["kv_len"] - s["q_start"].diff()
    live = i < s["keep_len"].long()[seq]
    seq, i, keep = seq[live], i[live], s["keep"].long()[live]
    src, dst = (_slots(s, seq, ctx.long()[seq] + j) for j in (keep, i))
    head = torch.arange(c["kv_heads"], device="cuda")[None]
    at = [(p[:, None], head, o[:, None]) if c["layout"] == "head" else (p[:, None], o[:, None], head) for p, o in (src, dst)]
    s["k"][at[1]] = s["k"][at[0]]
    s["v"][at[1]] = s["v"][at[0]]
    return {"k": s["k"], "v": s["v"], "length": ctx + s["keep_len"]}


# ------------------------------------------------------------------ the library's calls
def _own(s):
    import p100_b200 as P
    c, op = s["case"], s["case"]["op"]
    if op == "mask":
        r = P.tree_mask(s["parent"], s["q_start"], s["kv_len"], s["words"])
        return {"mask": r.mask, "position": r.position}
    if "desc" not in s:
        dim, kv_heads = c.get("dim", 128), c.get("kv_heads", 1)
        tokens_first = c.get("layout") == "token"
        s["desc"] = P.PagedDesc(
            n_seq=c["n_seq"], n_tokens=s["n_tokens"], max_q=s["max_q"], n_head_q=c.get("heads", kv_heads),
            n_head_kv=kv_heads, head_dim=dim, dtype=P.BF16 if c.get("dtype") == "bf16" else P.F16, page_size=c["page"],
            n_pages=s["n_pages"], max_pages=s["table"].shape[1], softcap=c.get("softcap", 0.0),
            head_stride=dim if tokens_first else 0, token_stride=kv_heads * dim if tokens_first else 0)
    if op == "plan":
        P.paged_plan(s["desc"], s["length"], s["none"], s["pool"], s["held"], s["table"])
        r = P.paged_plan(s["desc"], s["length"], s["n_new"], s["pool"], s["held"], s["table"])
        return {"q_start": r.q_start, "kv_len": r.kv_len, "slot": r.slot, "position": r.position, "table": s["table"],
                "held": s["held"], "pool": s["pool"]}
    where = (s["table"], s["q_start"], s["kv_len"])
    if op == "append":
        if "rope" not in s:
            kind = {"none": P.ROPE_NONE, "linear": P.ROPE_LINEAR, "ntk": P.ROPE_NTK, "bands": P.ROPE_BANDS,
                    "yarn": P.ROPE_YARN, "divisors": P.ROPE_DIVISORS}[c["scaling"]]
            s["rope"] = P.Rope(c["rope_dim"], THETA, half=c["half"], scaling=kind, **s["scaling"])
        q = P.paged_append_rope(s["desc"], s["qkv"], s["rope"], *where, s["k"], s["v"], position=s["position"],
                                q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
        return {"q": q, "k": s["k"], "v": s["v"]}
    if op == "keep":
        length = P.paged_keep(s["desc"], s["k"], s["v"], s["keep"], s["keep_len"], *where)
        return {"k": s["k"], "v": s["v"], "length": length}
    if "ws" not in s:
        s["ws"] = P.fa_paged_workspace(s["desc"])
    o, lse = P.fa_tree(s["desc"], s["q"], s["k"], s["v"], s["mask"], *where, ws=s["ws"])
    return {"o": o, "lse": lse}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "plan":
        _plain_plan(state, state["none"])
        return _plain_plan(state, state["n_new"])
    return {"mask": _plain_mask, "append": _plain_append, "attend": _plain_attend, "keep": _plain_keep}[op](state)


# ------------------------------------------------------------------ 64 bits
def _exact_append(s):
    c = s["case"]
    heads, kv_heads, dim, page, r = c["heads"], c["kv_heads"], c["dim"], c["page"], c["rope_dim"]
    q_start, kv_len, a = s["q_start"].tolist(), s["kv_len"].tolist(), s["scaling"]
    turn, gain = [], a.get("mscale", 1.0)   # radians a token, pair by pair
    for i in range(r // 2):
        base = THETA
        if c["scaling"] == "ntk":
            base *= a["factor"] ** (r / (r - 2))
        w = base ** (-2.0 * i / r)
        if c["scaling"] == "linear":
            w /= a["factor"]
        elif c["scaling"] == "bands":
            length = 2 * math.pi / w
            if length > a["original"] / a["low"]:
                w /= a["factor"]
            elif length > a["original"] / a["high"]:
                part = (a["original"] / length - a["low"]) / (a["high"] - a["low"])
                w = (1 - part) * w / a["factor"] + part * w
        elif c["scaling"] == "yarn":
            first, last = (r * math.log(a["original"] / (b * 2 * math.pi)) / (2 * math.log(THETA))
                           for b in (a["high"], a["low"]))
            first, last = max(math.floor(first), 0), min(math.ceil(last), r - 1)
            part = min(1.0, max(0.0, (i - first) / (last - first if last > first else 0.001)))
            w = w / a["factor"] * part + w * (1 - part)
            gain = 1 + 0.1 * math.log(a["factor"])
        elif c["scaling"] == "divisors":
            w /= a["divisors"][i]
        turn.append(w)
    turn = torch.tensor(turn, dtype=torch.float64, device="cuda")
    k_out, v_out = s["k"].double(), s["v"].double()
    if c["layout"] == "token":
        k_out, v_out = k_out.transpose(1, 2).contiguous(), v_out.transpose(1, 2).contiguous()
    queries = []
    for b in range(c["n_seq"]):
        lo, hi = q_start[b], q_start[b + 1]
        x = s["qkv"][lo:hi].double().view(-1, heads + 2 * kv_heads, dim)
        cell = torch.arange(kv_len[b] - (hi - lo), kv_len[b], device="cuda")
        at = cell if s["position"] is None else s["position"][lo:hi]
        spin = torch.polar(torch.full((hi - lo, r // 2), gain, dtype=torch.float64, device="cuda"),
                           at.double()[:, None] * turn)[:, None]
        done = []
        for part, w in ((x[:, :heads], s["q_norm"]), (x[:, heads:heads + kv_heads], s["k_norm"])):
            if w is not None:
                part = part / (part.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt() * w.double()
            z = part[..., :r]
            z = z.unflatten(-1, (2, r // 2)).transpose(-1, -2) if c["half"] else z.unflatten(-1, (r // 2, 2))
            y = torch.view_as_real(torch.view_as_complex(z.contiguous()) * spin)
            done.append(torch.cat([(y.transpose(-1, -2) if c["half"] else y).flatten(-2), part[..., r:]], -1))
        queries.append(done[0])
        slot = s["table"][b].long()[cell // page]
        k_out[slot, :, cell % page] = done[1]
        v_out[slot, :, cell % page] = x[:, heads + kv_heads:]
    if c["layout"] == "token":
        k_out, v_out = k_out.transpose(1, 2).contiguous(), v_out.transpose(1, 2).contiguous()
    return {"q": torch.cat(queries), "k": k_out, "v": v_out}


def _exact_attend(s):
    c = s["case"]
    heads, kv_heads, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    group = heads // kv_heads
    q_start, kv_len = s["q_start"].tolist(), s["kv_len"].tolist()
    words = s["mask"].cpu().numpy().view(np.uint8)
    bits = torch.from_numpy(np.unpackbits(words, axis=1, bitorder="little").astype(bool)).cuda()
    o = torch.zeros(s["n_tokens"], heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["n_tokens"], heads, dtype=torch.float64, device="cuda")
    for b in range(c["n_seq"]):
        t, lo, hi = kv_len[b], q_start[b], q_start[b + 1]
        where = torch.arange(t, device="cuda")
        slot, off = s["table"][b].long()[where // page], where % page
        sees = torch.ones(hi - lo, t, dtype=torch.bool, device="cuda")
        sees[:, t - (hi - lo):] = bits[lo:hi, :hi - lo]
        for h in range(kv_heads):
            k, v = ((x[slot, h, off] if c["layout"] == "head" else x[slot, off, h]).double() for x in (s["k"], s["v"]))
            for g in range(h * group, (h + 1) * group):
                y = s["q"][lo:hi, g].double() @ k.T / dim ** 0.5
                if c["softcap"]:
                    y = torch.tanh(y / c["softcap"]) * c["softcap"]
                y = torch.where(sees, y, -math.inf)
                lse[lo:hi, g] = torch.logsumexp(y, -1)
                o[lo:hi, g] = torch.softmax(y, -1) @ v
    return {"o": o, "lse": lse}


def exact(case, seed):
    if case["op"] not in ("append", "attend"):   # whole numbers and copies
        return None
    s = prepare(case, seed)
    return _exact_append(s) if case["op"] == "append" else _exact_attend(s)
