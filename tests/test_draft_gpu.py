"""Steps and drafted trees over the paged cache on the GPU: p100_paged_plan, p100_tree_mask, p100_paged_append_rope,
p100_fa_tree and p100_paged_keep against plain restatements, alone and as a step uses them together.

Tolerances.  Append: as test_paged_gpu's, the angles' error (2^-25 of a half turn from rounding, 2 units in the last
place of sine and cosine) being below 2^-21 of the pair's length, inside its 2^-18.  Attention: test_paged_gpu's bound,
which allows each probability one rounding of the 16-bit type."""
import math

import numpy as np
import pytest

import p100_b200 as P
from test_paged_gpu import Batch, check, near, types

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ plan
class Pool:
    """The plan on the host: a stack of free pages, each request's pages as a list."""

    def __init__(self, n_seq, n_pages):
        self.free = list(range(n_pages - 1, -1, -1))
        self.pages = [[] for _ in range(n_seq)]

    def step(self, length, n_new, page):
        need = [-(-(a + b) // page) for a, b in zip(length, n_new)]
        back = [p for own, n in zip(self.pages, need) for p in own[n:]]
        take = sum(max(0, n - len(own)) for own, n in zip(self.pages, need))
        if take > len(back) + len(self.free):
            return take - len(back) - len(self.free)
        self.free += back[::-1]   # the first one given back is the next one taken
        for own, n in zip(self.pages, need):
            del own[n:]
            while len(own) < n:
                own.append(self.free.pop())
        return 0


def plan_state(torch, n_seq, n_tokens, page, n_pages, max_pages):
    d = P.PagedDesc(n_seq=n_seq, n_tokens=n_tokens, n_head_q=1, n_head_kv=1, page_size=page, n_pages=n_pages,
                    max_pages=max_pages)
    return d, P.paged_pool(d)


def plan_check(torch, host, d, state, length, n_new, page, out=None):
    pool, held, table = state
    before = [list(p) for p in host.pages]
    missing = host.step(length, n_new, page)
    dev = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (length, n_new)]
    r = P.paged_plan(d, *dev, pool, held, table, out=out)
    P.check(P.device_error())
    start = np.zeros(len(length) + 1, np.int64) if missing else np.concatenate([[0], np.cumsum(n_new)])
    assert pool[1].item() == missing and pool[0].item() == len(host.free)
    assert r.q_start.tolist() == start.tolist()
    assert r.kv_len.tolist() == [a + (0 if missing else b) for a, b in zip(length, n_new)]
    assert pool[2:2 + len(host.free)].tolist() == host.free
    want = np.full((len(length), d.max_pages), -1)
    for s, p in enumerate(before if missing else host.pages):
        want[s, :len(p)] = p
    assert np.array_equal(table.cpu().numpy(), want)
    assert held.tolist() == [len(p) for p in host.pages]
    slot, position = np.full(d.n_tokens, -1), np.full(d.n_tokens, -1)
    if not missing:
        for s, (a, b) in enumerate(zip(length, n_new)):
            at = np.arange(a, a + b)
            position[start[s]:start[s] + b] = at
            slot[start[s]:start[s] + b] = [host.pages[s][t // page] * page + t % page for t in at]
    assert r.slot.tolist() == slot.tolist() and r.position.tolist() == position.tolist()
    return missing


@pytest.mark.parametrize("n_seq,draft,page,ctx", [(1, 1, 1, 5), (3, 7, 16, 100), (33, 4, 7, 60), (256, 1, 16, 900),
                                                  (257, 40, 24, 300), (1000, 16, 64, 500), (1024, 3, 5, 40)])
def test_plan(cuda, n_seq, draft, page, ctx):
    """Requests that grow, give drafts back, end and begin, over twelve steps; then the same step again."""
    rng = np.random.RandomState(n_seq)
    max_pages = -(-(ctx + draft) // page)
    d, state = plan_state(cuda, n_seq, n_seq * draft + 5, page, n_seq * max_pages, max_pages)
    host = Pool(n_seq, n_seq * max_pages)
    length = np.zeros(n_seq, np.int64)
    for _ in range(12):
        n_new = rng.randint(0, draft + 1, n_seq)
        plan_check(cuda, host, d, state, length.tolist(), n_new.tolist(), page)
        plan_check(cuda, host, d, state, length.tolist(), n_new.tolist(), page)
        length = length + (rng.rand(n_seq) * (n_new + 1)).astype(np.int64)
        length[rng.rand(n_seq) < 0.1] = 0
        length = np.where(rng.rand(n_seq) < 0.2, np.minimum(length, rng.randint(0, ctx + 1, n_seq)), length)
        grown = rng.rand(n_seq) < 0.2   # a prompt written elsewhere, as long as its pages allow
        length = np.where(grown, rng.randint(0, ctx + 1, n_seq), np.minimum(length, ctx))


def test_plan_undone_leaves_the_pool_as_it_was(cuda):
    d, state = plan_state(cuda, 40, 400, 8, 400, 10)
    host = Pool(40, 400)
    rng = np.random.RandomState(0)
    length = rng.randint(0, 60, 40)
    plan_check(cuda, host, d, state, length.tolist(), [0] * 40, 8)
    before = [x.clone() for x in state]
    plan_check(cuda, host, d, state, length.tolist(), rng.randint(0, 10, 40).tolist(), 8)
    plan_check(cuda, host, d, state, length.tolist(), [0] * 40, 8)
    for x, y in zip(state[1:], before[1:]):
        assert cuda.equal(x, y)
    n = int(before[0][0])
    assert cuda.equal(state[0][:2 + n], before[0][:2 + n])


def test_plan_without_enough_pages(cuda):
    """Nothing moves, no request has new tokens; the same requests fit when one gives its pages back."""
    d, state = plan_state(cuda, 3, 50, 4, 10, 10)
    host = Pool(3, 10)
    assert plan_check(cuda, host, d, state, [16, 8, 0], [0, 0, 0], 4) == 0
    assert plan_check(cuda, host, d, state, [16, 8, 0], [4, 4, 17], 4) == 3
    assert plan_check(cuda, host, d, state, [16, 8, 0], [1, 0, 16], 4) == 1
    assert plan_check(cuda, host, d, state, [0, 8, 0], [0, 4, 17], 4) == 0


@pytest.mark.parametrize("length,n_new,why", [([-1, 2], [1, 1], "negative length"), ([1, 2], [1, -1], "negative draft"),
                                              ([1, 30], [1, 11], "more than max_pages pages"),
                                              ([1, 2], [20, 11], "more than n_tokens")])
def test_plan_reports_bad_lengths(cuda, length, n_new, why):
    torch = cuda
    d, (pool, held, table) = plan_state(torch, 2, 30, 4, 40, 10)
    dev = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (length, n_new)]
    before = [x.clone() for x in (pool, held, table)]
    r = P.paged_plan(d, *dev, pool, held, table)
    with pytest.raises(P.InvalidArgument):
        P.check(P.device_error())
    assert pool[1].item() == -1 and r.q_start.tolist() == [0, 0, 0] and r.kv_len.tolist() == length
    assert bool((r.slot == -1).all()) and bool((r.position == -1).all())
    before[0][1] = -1
    assert all(torch.equal(x, y) for x, y in zip((pool, held, table), before))


@pytest.mark.parametrize("what", ["held", "count"])
def test_plan_reports_a_bad_state(cuda, what):
    torch = cuda
    d, (pool, held, table) = plan_state(torch, 2, 30, 4, 6, 5)
    if what == "held":
        held[1] = 6
    else:
        pool[0] = 7
    one = torch.ones(2, dtype=torch.int32, device="cuda")
    r = P.paged_plan(d, one, one, pool, held, table)
    with pytest.raises(P.InvalidArgument):
        P.check(P.device_error())
    assert pool[1].item() == -1 and r.q_start.tolist() == [0, 0, 0]


def test_plan_without_slots_and_into_given_tensors(cuda):
    torch = cuda
    d, (pool, held, table) = plan_state(torch, 2, 9000, 4, 5000, 2500)
    host = Pool(2, 5000)
    out = P.PagedPlan(*(torch.full((n,), 77, dtype=t, device="cuda")
                        for n, t in ((3, torch.int32), (2, torch.int32), (9000, torch.int64), (9000, torch.int32))))
    plan_check(torch, host, d, (pool, held, table), [7, 999], [8000, 1], 4, out)
    two = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
    r = P.paged_plan(d, two, two, pool, held, table, out=P.PagedPlan(out.q_start, out.kv_len, None, None))
    P.check(P.device_error())
    assert r.q_start.tolist() == [0, 3, 3] and r.kv_len.tolist() == [6, 0] and held.tolist() == [2, 0]


# ------------------------------------------------------------------ trees
def random_tree(rng, n, kind):
    if kind == "chain":
        return np.arange(-1, n - 1)
    if kind == "roots":
        return np.full(n, -1)
    return np.array([rng.randint(-1, i) if kind == "any" else max(-1, i - 1 - rng.randint(0, 4)) for i in range(n)])


def mask_of(parents, words):
    """(words of the masks, depths) of trees one behind another."""
    rows, depth = [], []
    for parent in parents:
        own = np.zeros((len(parent), len(parent)), bool)
        for i, p in enumerate(parent):
            if p >= 0:
                own[i] = own[p]
            own[i, i] = True
            depth.append(int(own[i].sum()) - 1)
        wide = np.zeros((len(parent), 32 * words), bool)
        wide[:, :len(parent)] = own
        rows.append(np.packbits(wide, axis=1, bitorder="little").view(np.int32))
    return np.concatenate(rows) if rows else np.zeros((0, words), np.int32), np.array(depth)


@pytest.mark.parametrize("sizes,kind,words", [([1], "any", 1), ([16], "any", 1), ([31, 32, 33], "any", 2),
                                              ([250] * 20, "near", 8), ([0, 5, 0, 64, 0], "any", 3),
                                              ([1024, 700], "chain", 32), ([1024], "roots", 32), ([1000, 3], "any", 32)])
def test_tree_mask(cuda, sizes, kind, words):
    torch = cuda
    rng = np.random.RandomState(len(sizes) + sizes[0])
    parents = [random_tree(rng, n, kind) for n in sizes]
    want, depth = mask_of(parents, words)
    lead, pad, total = 2, 3, sum(sizes)
    kv = [n + int(rng.randint(0, 5000)) for n in sizes]
    flat = np.concatenate([np.full(lead, 99)] + parents + [np.full(pad, 99)]).astype(np.int32)
    q_start = torch.from_numpy((lead + np.concatenate([[0], np.cumsum(sizes)])).astype(np.int32)).cuda()
    mask = torch.full((total + lead + pad, words), 7, dtype=torch.int32, device="cuda")
    position = torch.full((total + lead + pad,), 7, dtype=torch.int32, device="cuda")
    r = P.tree_mask(torch.from_numpy(flat).cuda(), q_start, torch.tensor(kv, dtype=torch.int32, device="cuda"), words,
                    mask, position)
    P.check(P.device_error())
    assert np.array_equal(r.mask[lead:lead + total].cpu().numpy(), want)
    base = np.repeat(np.array(kv) - np.array(sizes), sizes)
    assert np.array_equal(r.position[lead:lead + total].cpu().numpy(), base + depth)
    for x in (mask, position):   # rows of no sequence
        assert bool((x[:lead] == 7).all()) and bool((x[lead + total:] == 7).all())


def test_tree_mask_reports_bad_trees(cuda):
    """A parent at or behind its child counts as -1; a tree too large for the words is left out."""
    torch = cuda
    i32 = dict(dtype=torch.int32, device="cuda")
    r = P.tree_mask(torch.tensor([-1, 1, 0, -7, 2], **i32), torch.tensor([0, 5], **i32), torch.tensor([9], **i32), 1)
    with pytest.raises(P.InvalidArgument):
        P.check(P.device_error())
    assert r.mask[:, 0].tolist() == [1, 2, 5, 8, 21] and r.position.tolist() == [4, 4, 5, 4, 6]
    mask = torch.full((40, 1), 7, **i32)
    for start, kv in (([0, 4, 37], [4, 90]), ([0, 4, 50], [4, 90]), ([0, 4, 3], [4, 90]), ([0, 4, 30], [4, 20])):
        mask.fill_(7)
        P.tree_mask(torch.full((40,), -1, **i32), torch.tensor(start, **i32), torch.tensor(kv, **i32), 1, mask)
        with pytest.raises(P.InvalidArgument):
            P.check(P.device_error())
        assert mask[:, 0].tolist() == [1, 2, 4, 8] + [7] * 36


# ------------------------------------------------------------------ append
def rope64(rope_kw, positions):
    """cos and sin of every position and pair as float64, the angles reduced in long double."""
    kw = dict(rope_kw)
    r, theta, kind = kw["rope_dim"], np.longdouble(kw["theta"]), kw.get("scaling", P.ROPE_NONE)
    i = np.arange(r // 2).astype(np.longdouble)
    if kind == P.ROPE_NTK:
        theta = theta * np.longdouble(kw["factor"]) ** (np.longdouble(r) / (r - 2))
    f = theta ** (-2 * i / r)
    pi = np.longdouble("3.14159265358979323846264338327950288")
    if kind == P.ROPE_LINEAR:
        f = f / kw["factor"]
    if kind == P.ROPE_BANDS:
        w = np.clip((kw["original"] * f / (2 * pi) - kw["low"]) / (kw["high"] - kw["low"]), 0, 1)
        f = w * f + (1 - w) * f / kw["factor"]
    if kind == P.ROPE_YARN:
        lo, hi = (r * np.log(kw["original"] / (b * 2 * pi)) / (2 * np.log(theta)) for b in (kw["high"], kw["low"]))
        lo, hi = max(np.floor(lo), 0), min(np.ceil(hi), r - 1)
        w = np.clip((i - lo) / (hi - lo if hi > lo else np.longdouble("0.001")), 0, 1)
        f = f / kw["factor"] * w + f * (1 - w)
    if kind == P.ROPE_DIVISORS:
        f = f / np.array(kw["divisors"], np.longdouble)
    m = kw.get("mscale", 0) or (0.1 * math.log(kw["factor"]) + 1 if kind == P.ROPE_YARN else 1.0)
    turns = np.asarray(positions).astype(np.longdouble)[:, None] * f / (2 * pi)
    angle = ((turns - np.floor(turns)) * 2 * pi).astype(np.float64)
    return np.cos(angle) * m, np.sin(angle) * m


def append64(b, qkv, rope_kw, half, positions, q_norm, k_norm, eps):
    """q and every sequence's k and v rows in 64 bits with the length that scales their FP32 error."""
    torch = b.torch
    r = rope_kw["rope_dim"]
    x = qkv.double().view(b.n_tokens, b.hq + 2 * b.hkv, b.dim).clone()
    cos, sin = (torch.from_numpy(t).cuda()[:, None] for t in rope64(rope_kw, positions))

    def turned(y, w):
        if w is not None:
            y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
        z = y[..., :r]
        a, c = (z[..., :r // 2], z[..., r // 2:]) if half else (z[..., 0::2], z[..., 1::2])
        t, size = (a * cos - c * sin, a * sin + c * cos), a.abs() + c.abs()
        t, size = (torch.cat(t, -1), torch.cat([size, size], -1)) if half else (
            torch.stack(t, -1).flatten(-2), torch.stack([size, size], -1).flatten(-2))
        return torch.cat([t, y[..., r:]], -1), torch.cat([size * float(cos.abs().max() + sin.abs().max()) / 2 + size,
                                                          y[..., r:].abs()], -1)

    return (turned(x[:, :b.hq], q_norm), turned(x[:, b.hq:b.hq + b.hkv], k_norm), x[:, b.hq + b.hkv:])


ROPES = [
    dict(theta=10000.0),
    dict(theta=500000.0, scaling=P.ROPE_LINEAR, factor=4.0),
    dict(theta=10000.0, scaling=P.ROPE_NTK, factor=8.0),
    dict(theta=500000.0, scaling=P.ROPE_BANDS, factor=8.0, low=1.0, high=4.0, original=8192),
    dict(theta=10000.0, scaling=P.ROPE_YARN, factor=16.0, low=1.0, high=32.0, original=4096),
    dict(theta=10000.0, scaling=P.ROPE_DIVISORS, mscale=1.25),
]
APPENDS = [
    # q_lens, kv_lens, hq, hkv, dim, src, dtype, page, layout, norm, rope_dim
    ([1], [1], 1, 1, 64, "f32", "f16", 1, "head", False, 64),
    ([8], [4096], 32, 8, 128, "f32", "f16", 16, "head", False, 64),
    ([5, 1, 33], [70, 1, 33], 6, 2, 128, "bf16", "bf16", 7, "token", True, 128),
    ([100, 0, 40], [163, 9, 1000], 8, 1, 64, "f16", "f16", 24, "head", True, 20),
    ([17], [40], 5, 5, 64, "f32", "bf16", 64, "token", True, 2 + 2),
    ([64, 3], [64, 130], 3, 1, 128, "f16", "bf16", 32, "head", False, 96),
    ([2] * 70, [3 + i for i in range(70)], 4, 2, 64, "bf16", "f16", 16, "head", False, 34),
    ([9, 30], [9, 300], 7, 7, 128, "bf16", "f16", 16, "token", True, 40),
    ([9, 30], [9, 300], 7, 7, 128, "f32", "bf16", 16, "head", False, 126),
]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append_rope(cuda, case, half):
    torch = cuda
    q_lens, kv_lens, hq, hkv, dim, src, dtype, page, layout, norm, rope_dim = APPENDS[case]
    b = Batch(torch, q_lens, kv_lens, hq, hkv, dim, dtype, page, layout, seed=50 + case, pad_rows=2, lead_rows=1)
    rng = np.random.RandomState(case)
    for given in (False, True):
        kw = dict(ROPES[(case + 3 * given + 2 * half) % len(ROPES)], rope_dim=rope_dim)
        if kw.get("scaling") == P.ROPE_DIVISORS:
            kw["divisors"] = [1.0 + i for i in range(rope_dim // 2)]
        own = np.concatenate([[0]] + [np.arange(t - n, t) for n, t in zip(q_lens, kv_lens)] + [[0, 0]])
        far = rng.randint(0, 1 << rng.randint(3, 31), b.n_tokens)
        positions = far if given else own
        qkv = (torch.randn(b.n_tokens, (hq + 2 * hkv) * dim, generator=b.gen, device="cuda") * 2).to(types(torch)[src][0])
        w = [torch.rand(dim, generator=b.gen, device="cuda") + 0.5 if norm else None for _ in range(2)]
        q = torch.full((b.n_tokens, hq, dim), 7.0, dtype=b.t, device="cuda")
        b.k.fill_(math.nan)
        b.v.fill_(math.nan)
        P.paged_append_rope(b.desc(), qkv, P.Rope(half=half, **kw), b.table, b.q_start, b.kv_len, b.k, b.v,
                            position=torch.from_numpy(far.astype(np.int32)).cuda() if given else None, q_norm=w[0],
                            k_norm=w[1], eps=1e-6, q=q)
        P.check(P.device_error())
        (want, length), (k, klen), v = append64(b, qkv, kw, half, positions, w[0], w[1], 1e-6)
        lo, hi = 1, b.n_tokens - 2
        assert bool((q[:lo] == 7).all()) and bool((q[hi:] == 7).all())
        near(torch, b.t, q[lo:hi], want[lo:hi], length[lo:hi])
        for s, n in enumerate(q_lens):
            at = slice(int(b.q_start_host[s]), int(b.q_start_host[s]) + n)
            first = kv_lens[s] - n
            near(torch, b.t, b.rows(b.k, s, first), k[at], klen[at])
            near(torch, b.t, b.rows(b.v, s, first), v[at], v[at].abs() * 0)
        for x in (b.k, b.v):   # every other row of the pages is as it was
            assert int((~torch.isnan(x)).sum()) == sum(q_lens) * hkv * dim


@pytest.mark.parametrize("half", [False, True])
def test_append_rope_keeps_the_rest_of_a_head(cuda, half):
    """Values behind rope_dim go through as they are, infinite ones too, and touch no rotated one."""
    torch = cuda
    for rope_dim, src in ((20, "f32"), (20, "bf16"), (64, "f16"), (48, "f32")):
        b = Batch(torch, [3], [3], 2, 1, 128, "f16", 16)
        qkv = torch.randn(3, 4 * 128, generator=b.gen, device="cuda").to(types(torch)[src][0])
        x = qkv.view(3, 4, 128)
        x[:, :, rope_dim:] = math.inf
        q = P.paged_append_rope(b.desc(), qkv, P.Rope(rope_dim, 10000.0, half=half), b.table, b.q_start, b.kv_len, b.k, b.v)
        P.check(P.device_error())
        k = b.rows(b.k, 0)
        assert bool(torch.isinf(q[:, :, rope_dim:]).all()) and bool(torch.isinf(k[:, :, rope_dim:]).all())
        assert bool(torch.isfinite(q[:, :, :rope_dim]).all()) and bool(torch.isfinite(k[:, :, :rope_dim]).all())


def test_append_rope_equals_the_table(cuda):
    """At small positions the computed angles give what p100_paged_append's table gives, to a rounding."""
    torch = cuda
    for half in (False, True):
        b = Batch(torch, [60], [100], 8, 2, 128, "f16", 16)
        qkv = torch.randn(60, 12 * 128, generator=b.gen, device="cuda")
        cs = torch.from_numpy(P.rope_table(100, 128, 500000.0)).cuda()
        where = (b.table, b.q_start, b.kv_len, b.k, b.v)
        q0 = P.paged_append(b.desc(), qkv, *where, rope_cs=cs, rope_half=half)
        k0 = b.k.clone()
        q1 = P.paged_append_rope(b.desc(), qkv, P.Rope(128, 500000.0, half=half), *where)
        P.check(P.device_error())
        for x, y in ((q0, q1), (k0, b.k)):
            live = ~torch.isnan(x)
            size = x[live].float().abs() + 2.0 ** -10
            assert bool(((x[live].float() - y[live].float()).abs() <= 2.0 ** -10 * size).all())


def test_append_rope_reports_bad_positions(cuda):
    torch = cuda
    b = Batch(torch, [4, 2], [4, 2], 2, 1, 64, "f16", 4)
    qkv = torch.randn(6, 4 * 64, device="cuda")
    position = torch.tensor([0, -1, 2, (1 << 31) - 1, 5, 6], dtype=torch.int32, device="cuda")
    q = torch.full((6, 2, 64), 7.0, dtype=torch.float16, device="cuda")
    P.paged_append_rope(b.desc(), qkv, P.Rope(64, 10000.0), b.table, b.q_start, b.kv_len, b.k, b.v, position=position, q=q)
    with pytest.raises(P.InvalidArgument):
        P.check(P.device_error())
    left = (q == 7).flatten(1).all(1)
    assert left.tolist() == [False, True, False, False, False, False]
    assert bool(torch.isnan(b.rows(b.k, 0)[1]).all()) and not bool(torch.isnan(b.rows(b.k, 0)[[0, 2, 3]]).any())


# ------------------------------------------------------------------ attention
def tree64(b, q, bits, scale=0.0, softcap=0.0):
    """attend64 of test_paged_gpu with the masks' bits [n_tokens, columns] in place of the causal ones."""
    torch = b.torch
    scale = scale or 1.0 / math.sqrt(b.dim)
    group, u = b.hq // b.hkv, torch.finfo(b.t).eps / 2
    o = torch.full((b.n_tokens, b.hq, b.dim), math.nan, dtype=torch.float64, device="cuda")
    lse = torch.full((b.n_tokens, b.hq), math.nan, dtype=torch.float64, device="cuda")
    tol_o, tol_l = torch.zeros_like(o), torch.zeros_like(lse)
    for s, (n, t) in enumerate(zip(b.q_lens, b.kv_lens)):
        if n == 0:
            continue
        lo = int(b.q_start_host[s])
        seen = torch.ones(n, t, dtype=torch.bool, device="cuda")
        seen[:, t - n:] = bits[lo:lo + n, :n]
        k, v = b.rows(b.k, s), b.rows(b.v, s)
        for h in range(b.hq):
            qh, kh, vh = q[lo:lo + n, h].double(), k[:, h // group], v[:, h // group]
            x = qh @ kh.T * scale
            err = b.dim * 2.0 ** -24 * abs(scale) * (qh.abs() @ kh.abs().T) + 2.0 ** -20
            if softcap:
                x = torch.tanh(x / softcap) * softcap
                err = err + 2.0 ** -20 * softcap
            x = torch.where(seen, x, torch.full_like(x, -math.inf))
            err = torch.where(seen, err, torch.zeros_like(err))
            m = x.amax(1, keepdim=True)
            p = torch.where(m > -math.inf, torch.exp(x - m.clamp(min=-1e30)), torch.zeros_like(x))
            total = p.sum(1, keepdim=True)
            p = torch.where(total > 0, p / total.clamp(min=1e-300), torch.zeros_like(p))
            e = err.amax(1, keepdim=True)
            o[lo:lo + n, h] = p @ vh
            lse[lo:lo + n, h] = (m + total.log())[:, 0]
            spread = p @ vh.abs()
            tiny = 2.0 ** -25 * vh.abs().sum(0) if b.t == torch.float16 else 0.0
            tol_o[lo:lo + n, h] = u * o[lo:lo + n, h].abs() + (u * (1 + u) + 2 * e + 2.0 ** -18) * spread + tiny + 2.0 ** -24
            tol_l[lo:lo + n, h] = e[:, 0] + 2.0 ** -18 * (1 + lse[lo:lo + n, h].abs().clamp(max=1e30))
    return o, lse, tol_o, tol_l


def masks(b, rng, kind, words):
    """(int32 words on the device, bits) of every row; rows of no sequence and bits behind a tree are set."""
    bits = np.ones((b.n_tokens, 32 * words), bool)
    for s, n in enumerate(b.q_lens):
        lo = int(b.q_start_host[s])
        if kind == "bits":
            bits[lo:lo + n] = rng.rand(n, 32 * words) < 0.4
        elif kind == "empty":
            bits[lo:lo + n, :n] = False
        else:
            own = mask_of([random_tree(rng, n, kind)], words)[0]
            bits[lo:lo + n, :n] = np.unpackbits(own.view(np.uint8), axis=1, bitorder="little")[:, :n]
    packed = np.packbits(bits, axis=1, bitorder="little").view(np.int32)
    return b.torch.from_numpy(packed).cuda(), b.torch.from_numpy(bits).cuda()


def attend_tree(b, q, mask, **kw):
    o, lse = P.fa_tree(b.desc(**kw), q, b.k, b.v, mask, b.table, b.q_start, b.kv_len)
    P.check(P.device_error())
    return o, lse


# lengths of one, trees without a context, tails over one to three tiles and pages
TREES = [
    # q_lens, kv_lens, hq, hkv, dim, dtype, page, layout, words
    ([1], [1], 1, 1, 64, "f16", 1, "head", 1),
    ([1, 1, 1], [63, 64, 129], 4, 2, 128, "bf16", 7, "token", 1),
    ([4, 2, 3], [4, 300, 127], 4, 1, 128, "f16", 16, "head", 1),
    ([16], [4096], 32, 8, 128, "f16", 16, "head", 1),
    ([5, 3, 1, 5], [3001, 129, 1, 5], 12, 4, 64, "f16", 24, "token", 1),
    ([8, 7, 8, 0, 2], [1000, 128, 8, 0, 2000], 64, 8, 128, "bf16", 64, "head", 2),
    ([17, 31, 32], [17, 255, 258], 1, 1, 128, "bf16", 33, "token", 1),
    ([33, 40], [160, 257], 6, 2, 64, "bf16", 16, "head", 3),
    ([64, 64, 20], [700, 64, 500], 32, 8, 128, "f16", 128, "head", 2),
    ([100], [2500], 8, 1, 128, "bf16", 9, "head", 4),      # 800 rows of one kv head
    ([129], [400], 3, 1, 64, "f16", 256, "token", 5),
    ([250, 130, 1], [260, 3000, 900], 5, 5, 128, "f16", 64, "head", 8),
    ([1000], [1100], 2, 1, 64, "bf16", 32, "head", 32),
    ([3 + i % 9 for i in range(60)], [20 + 37 * i for i in range(60)], 8, 2, 128, "f16", 16, "token", 1),
    ([2] * 130, [2 + 9 * i for i in range(130)], 40, 40, 64, "bf16", 48, "head", 1),
    ([20, 9], [6000, 9000], 24, 1, 128, "bf16", 1, "head", 1),
]


@pytest.mark.parametrize("kind", ["any", "bits", "chain"])
@pytest.mark.parametrize("case", range(len(TREES)))
def test_tree_attention(cuda, case, kind):
    q_lens, kv_lens, hq, hkv, dim, dtype, page, layout, words = TREES[case]
    b = Batch(cuda, q_lens, kv_lens, hq, hkv, dim, dtype, page, layout, seed=case, pad_rows=2, lead_rows=1)
    b.fill()
    q = b.queries()
    mask, bits = masks(b, np.random.RandomState(case), kind, words)
    check(cuda, b, *attend_tree(b, q, mask), tree64(b, q, bits))


@pytest.mark.parametrize("q_lens,kv_lens,hq,hkv", [([4, 4], [400, 4], 4, 1), ([30, 7], [400, 9], 8, 2)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_tree_softcap_scale_fp32_and_empty_rows(cuda, q_lens, kv_lens, hq, hkv, dtype):
    """Capped and negatively scaled scores, unrounded outputs, rows that see nothing of the tree (and, without a
    context, nothing at all)."""
    b = Batch(cuda, q_lens, kv_lens, hq, hkv, 128, dtype, 16, seed=3)
    b.fill()
    q = b.queries(4.0)
    for kind in ("any", "empty", "bits"):
        mask, bits = masks(b, np.random.RandomState(1), kind, 2)
        for kw in (dict(softcap=20.0, scale=0.2), dict(scale=-0.15), dict(scale=-0.15, softcap=20.0), {}):
            want = tree64(b, q, bits, **kw)
            check(cuda, b, *attend_tree(b, q, mask, **kw), want)
            o, lse = attend_tree(b, q, mask, o_fp32=True, causal=False, **kw)
            assert o.dtype == cuda.float32
            check(cuda, b, o, lse, want)


@pytest.mark.parametrize("q_lens,kv_lens", [([0, 0], [5, 0]), ([3, 0, 2], [3, 7, 2]), ([40, 0, 2], [40, 7, 90])])
def test_tree_without_context(cuda, q_lens, kv_lens):
    """Trees that are the whole sequence, with masks that name nothing: o = 0, lse = -inf."""
    b = Batch(cuda, q_lens, kv_lens, 4, 2, 64, "bf16", 8, pad_rows=3)
    b.fill()
    q = b.queries()
    for kind in ("empty", "any"):
        mask, bits = masks(b, np.random.RandomState(0), kind, 2)
        o = cuda.full((b.n_tokens, 4, 64), 7.0, dtype=b.t, device="cuda")
        lse = cuda.full((b.n_tokens, 4), 7.0, device="cuda")
        P.fa_tree(b.desc(), q, b.k, b.v, mask, b.table, b.q_start, b.kv_len, o=o, lse=lse)
        P.check(P.device_error())
        check(cuda, b, o, lse, tree64(b, q, bits))
        end = sum(q_lens)
        assert bool((o[end:] == 7).all()) and bool((lse[end:] == 7).all())


@pytest.mark.parametrize("q_lens,kv_lens", [([5, 1], [300, 77]), ([64, 20], [700, 20])])
def test_chain_is_causal_attention(cuda, q_lens, kv_lens):
    b = Batch(cuda, q_lens, kv_lens, 8, 4, 128, "f16", 16)
    b.fill()
    q = b.queries()
    mask, _ = masks(b, None, "chain", 2)
    o, lse = attend_tree(b, q, mask, o_fp32=True)
    o1, lse1 = P.fa_paged(b.desc(o_fp32=True), q, b.k, b.v, b.table, b.q_start, b.kv_len)
    # each is within 2^-11 of sum p |v| (values up to 5) of the other's probabilities
    assert bool(((o - o1).abs() <= 5 * 2.0 ** -10).all()) and bool(((lse - lse1).abs() <= 2.0 ** -16 * (1 + lse.abs())).all())


@pytest.mark.parametrize("dim,group", [(64, 4), (128, 2), (128, 8)])
def test_tree_without_pages(cuda, dim, group):
    """A cache without a page: trees whose masks are empty in sequences of no length give 0 and -inf."""
    torch = cuda
    d = P.PagedDesc(n_seq=2, n_tokens=7, max_q=4, n_head_q=2 * group, n_head_kv=2, page_size=16, n_pages=0, max_pages=1,
                    head_dim=dim)
    i32 = dict(dtype=torch.int32, device="cuda")
    k = torch.zeros(8, dtype=torch.float16, device="cuda")
    q = torch.ones(7, 2 * group, dim, dtype=torch.float16, device="cuda")
    o, lse = P.fa_tree(d, q, k, k, torch.full((7, 1), -1, **i32), torch.full((2, 1), -1, **i32), torch.tensor([0, 3, 7], **i32),
                       torch.zeros(2, **i32))
    P.check(P.device_error())
    assert bool((o == 0).all()) and bool(torch.isneginf(lse).all())


def test_tree_reports_too_many_tokens(cuda):
    b = Batch(cuda, [33, 2], [50, 60], 4, 1, 64, "f16", 16)
    b.fill()
    q = b.queries()
    mask = cuda.full((b.n_tokens, 1), -1, dtype=cuda.int32, device="cuda")
    o = cuda.full((b.n_tokens, 4, 64), 7.0, dtype=b.t, device="cuda")
    P.fa_tree(b.desc(), q, b.k, b.v, mask, b.table, b.q_start, b.kv_len, o=o)
    with pytest.raises(P.InvalidArgument):
        P.check(P.device_error())
    assert bool((o == 7).all())


# ------------------------------------------------------------------ keep
KEEPS = [
    # q_lens, kv_lens, hkv, dim, page, layout
    ([1], [1], 1, 64, 1, "head"),
    ([8], [4096], 8, 128, 16, "head"),
    ([64, 1, 0, 33], [64, 900, 7, 100], 5, 128, 24, "token"),
    ([200, 40], [1000, 40], 3, 64, 7, "head"),
    ([20] * 100, [20 + 3 * i for i in range(100)], 2, 128, 64, "token"),
]


@pytest.mark.parametrize("part", [0.0, 0.3, 0.8, 1.0])
@pytest.mark.parametrize("case", range(len(KEEPS)))
def test_keep(cuda, case, part):
    torch = cuda
    q_lens, kv_lens, hkv, dim, page, layout = KEEPS[case]
    b = Batch(torch, q_lens, kv_lens, 2 * hkv, hkv, dim, "bf16", page, layout, seed=case, pad_rows=2, lead_rows=1)
    b.fill()
    rng = np.random.RandomState(case)
    keep = np.full(b.n_tokens, -9, np.int32)
    lists = []
    for s, n in enumerate(q_lens):
        own = np.flatnonzero(rng.rand(n) < part)
        keep[b.q_start_host[s]:b.q_start_host[s] + len(own)] = own
        lists.append(own)
    want = []
    for x in (b.k, b.v):
        y = x.clone()
        for s, own in enumerate(lists):
            page_at, off = b.slots(s, kv_lens[s] - q_lens[s])
            own = torch.from_numpy(own).cuda()
            n = len(own)
            if layout == "head":
                y[page_at[:n], :, off[:n]] = x[page_at[own], :, off[own]]
            else:
                y[page_at[:n], off[:n]] = x[page_at[own], off[own]]
        want.append(y)
    i32 = dict(dtype=torch.int32, device="cuda")
    length = P.paged_keep(b.desc(), b.k, b.v, torch.from_numpy(keep).cuda(), torch.tensor([len(x) for x in lists], **i32),
                          b.table, b.q_start, b.kv_len)
    P.check(P.device_error())
    assert length.tolist() == [t - n + len(x) for n, t, x in zip(q_lens, kv_lens, lists)]
    for x, y in zip((b.k, b.v), want):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))


def test_keep_reports_bad_lists(cuda):
    """Counts out of range leave the sequence out, indices out of order their row."""
    torch = cuda
    i32 = dict(dtype=torch.int32, device="cuda")
    b = Batch(torch, [4, 4], [20, 30], 2, 2, 64, "f16", 8)
    b.fill()
    for keep, count, moved in (([0, 1, 2, 3, 1, 3, 0, 0], [5, 2], [(1, 0, 1), (1, 1, 3)]),
                               ([0, 1, 2, 3, 1, 3, 0, 0], [-1, 2], [(1, 0, 1), (1, 1, 3)]),
                               ([2, 1, 3, 0, 3, 4, 0, 0], [3, 2], [(0, 0, 2), (0, 2, 3), (1, 0, 3)]),
                               ([-1, 3, 3, 0, 0, 0, 0, 0], [3, 0], [(0, 1, 3)])):
        k, v = b.k.clone(), b.v.clone()
        want = k.clone()
        for s, i, j in moved:
            page_at, off = b.slots(s, b.kv_lens[s] - 4)
            want[page_at[i], :, off[i]] = k[page_at[j], :, off[j]]
        P.paged_keep(b.desc(), k, v, torch.tensor(keep, **i32), torch.tensor(count, **i32), b.table, b.q_start, b.kv_len)
        with pytest.raises(P.InvalidArgument):
            P.check(P.device_error())
        live = ~torch.isnan(want)
        assert torch.equal(k[live], want[live])
    table = b.table.clone()
    table[0, 2] = b.n_pages   # the page of the last new tokens
    k = b.k.clone()
    P.paged_keep(b.desc(), k, b.v.clone(), torch.tensor([1, 2, 3, 0, 0, 0, 0, 0], **i32), torch.tensor([3, 0], **i32), table,
                 b.q_start, b.kv_len)
    with pytest.raises(P.InvalidArgument):
        P.check(P.device_error())
    live = ~torch.isnan(b.k)
    assert torch.equal(k[live], b.k[live])


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("hq,hkv,dim,dtype", [(8, 2, 64, "f16"), (16, 2, 128, "bf16")])
def test_steps_together(cuda, hq, hkv, dim, dtype):
    """Drafts accepted in part over six steps by one captured graph, a plan to a plan: what the cache then holds and what
    the last drafts attend to are those of the accepted tokens laid out densely."""
    torch = cuda
    n_seq, draft, page, steps, words = 5, 9, 8, 6, 1
    t, kind = types(torch)[dtype]
    i32 = dict(dtype=torch.int32, device="cuda")
    d = P.PagedDesc(n_seq=n_seq, n_tokens=n_seq * draft, max_q=draft, n_head_q=hq, n_head_kv=hkv, page_size=page,
                    n_pages=n_seq * 9, max_pages=8, head_dim=dim, dtype=kind)
    pool, held, table = P.paged_pool(d)
    shape = (d.n_pages, hkv, page, dim)
    k, v = torch.zeros(shape, dtype=t, device="cuda"), torch.zeros(shape, dtype=t, device="cuda")
    rope = P.Rope(dim // 2, 10000.0, half=True, scaling=P.ROPE_LINEAR, factor=2.0)
    ws = P.fa_paged_workspace(d)
    length, n_new = torch.zeros(n_seq, **i32), torch.zeros(n_seq, **i32)
    parent, keep, keep_len = torch.zeros(n_seq * draft, **i32), torch.zeros(n_seq * draft, **i32), torch.zeros(n_seq, **i32)
    qkv = torch.zeros(n_seq * draft, (hq + 2 * hkv) * dim, dtype=t, device="cuda")

    def step():
        plan = P.paged_plan(d, length, n_new, pool, held, table)
        tree = P.tree_mask(parent, plan.q_start, plan.kv_len, words)
        q = P.paged_append_rope(d, qkv, rope, table, plan.q_start, plan.kv_len, k, v, position=tree.position)
        o, lse = P.fa_tree(d, q, k, v, tree.mask, table, plan.q_start, plan.kv_len, ws=ws)
        P.paged_keep(d, k, v, keep, keep_len, table, plan.q_start, plan.kv_len, length=length)
        return plan, tree, q, o, lse

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):   # nothing new: every kernel runs once before the capture
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, tree, q, o, lse = step()
    rng = np.random.RandomState(hq)
    rows = [[[], []] for _ in range(n_seq)]   # accepted k and v rows
    for _ in range(steps):
        sizes = rng.randint(1, draft + 1, n_seq)
        parents = [random_tree(rng, n, "any") for n in sizes]
        paths = []
        for p in parents:   # the way to a random token of the tree
            at, path = int(rng.randint(0, len(p))), []
            while at >= 0:
                path.append(at)
                at = int(p[at])
            paths.append(path[::-1])
        flat = lambda lists: torch.tensor(np.concatenate(lists).tolist(), **i32)   # noqa: E731
        n_new.copy_(torch.tensor(sizes.tolist(), **i32))
        parent[:sizes.sum()] = flat(parents)
        keep.fill_(-1)
        start = np.concatenate([[0], np.cumsum(sizes)])
        for s, path in enumerate(paths):
            keep[start[s]:start[s] + len(path)] = torch.tensor(path, **i32)
        keep_len.copy_(torch.tensor([len(p) for p in paths], **i32))
        qkv.copy_(torch.randn(qkv.shape, device="cuda").to(t))
        before = [len(r[0]) for r in rows]
        graph.replay()
        P.check(P.device_error())
        assert length.tolist() == [a + len(p) for a, p in zip(before, paths)]
        # the step's tokens in 64 bits: rotation at the depth, then attention to the accepted rows and the ancestors
        depth = mask_of(parents, words)[1]
        positions = np.repeat(before, sizes) + depth
        assert tree.position[:sizes.sum()].tolist() == positions.tolist()
        cos, sin = (torch.from_numpy(x).cuda()[:, None] for x in rope64(
            dict(rope_dim=dim // 2, theta=10000.0, scaling=P.ROPE_LINEAR, factor=2.0), positions))
        x = qkv[:sizes.sum()].double().view(-1, hq + 2 * hkv, dim)

        def turned(y):
            a, c = y[..., :dim // 4], y[..., dim // 4:dim // 2]
            return torch.cat([a * cos - c * sin, a * sin + c * cos, y[..., dim // 2:]], -1).to(t).double()

        qt, kt, vt = turned(x[:, :hq]), turned(x[:, hq:hq + hkv]), x[:, hq + hkv:]
        group = hq // hkv
        for s in range(n_seq):
            for i in range(sizes[s]):
                way, at = [], i
                while at >= 0:
                    way.append(start[s] + at)
                    at = int(parents[s][at])
                kk = torch.stack(rows[s][0] + [kt[w] for w in way])
                vv = torch.stack(rows[s][1] + [vt[w] for w in way])
                y = torch.einsum("hd,thd->ht", qt[start[s] + i], kk.repeat_interleave(group, 1)) / dim ** 0.5
                want = torch.einsum("ht,thd->hd", torch.softmax(y, 1), vv.repeat_interleave(group, 1))
                # the queries' and keys' roundings may fall the other way (one step of the type): 2^-7 of a score's terms
                u = torch.finfo(t).eps / 2
                tol = u * want.abs() + 4 * u * vv.abs().amax() * (1 + (qt[start[s] + i].abs().amax() * kk.abs().sum(-1).amax()) / dim ** 0.5)
                assert bool(((o[start[s] + i].double() - want).abs() <= tol).all())
            rows[s][0] += [kt[start[s] + i] for i in paths[s]]
            rows[s][1] += [vt[start[s] + i] for i in paths[s]]
        cache = table.cpu().numpy()
        for s in range(n_seq):
            at = np.arange(len(rows[s][0]))
            page_at = torch.from_numpy(cache[s][at // page].astype(np.int64)).cuda()
            off = torch.from_numpy(at % page).cuda()
            got = k[page_at, :, off].double()
            want = torch.stack(rows[s][0])
            assert bool(((got - want).abs() <= torch.finfo(t).eps * want.abs() + 2.0 ** -16).all())
            assert torch.equal(v[page_at, :, off].double(), torch.stack(rows[s][1]))
