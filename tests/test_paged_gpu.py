"""The paged cache on the GPU: p100_paged_append and p100_fa_paged against 64-bit restatements.

Tolerances.  u = eps / 2 of the 16-bit type (a rounding to nearest is off by at most u relative).
Append: one rounding of an FP32 result whose relative error (a sum of 128 squares, a division, four products) is
below 2^-18 of the pair's length.  Attention: the output's rounding, u |o|; each probability's rounding, u sum p |v|
(p normalised); in float16, probabilities below 2^-14 lose at most 2^-25 of the largest; FP32 scores, off by at most
D 2^-24 scale sum |q k|, which moves p by that factor (twice: numerator and sum), and 2^-18 for the exponentials and
sums.  lse: the scores' error and 2^-18 (1 + |lse|)."""
import math

import numpy as np
import pytest

import p100_b200 as P

pytestmark = pytest.mark.gpu


def types(torch):
    return {"f16": (torch.float16, P.F16), "bf16": (torch.bfloat16, P.BF16), "f32": (torch.float32, P.F32)}


class Batch:
    """Sequences of new tokens over a paged cache with shuffled pages; whatever no sequence holds is NaN."""

    def __init__(self, torch, q_lens, kv_lens, hq, hkv, dim, dtype="f16", page=16, layout="head", seed=0, spare=2,
                 pad_rows=0, lead_rows=0):
        self.torch, self.hq, self.hkv, self.dim, self.page, self.layout = torch, hq, hkv, dim, page, layout
        self.q_lens, self.kv_lens = list(q_lens), list(kv_lens)
        self.t, self.kind = types(torch)[dtype]
        rng = np.random.RandomState(seed)
        g = torch.Generator(device="cuda")
        g.manual_seed(seed + 1)
        self.gen = g
        n = len(q_lens)
        self.lead = lead_rows
        self.n_tokens = sum(q_lens) + pad_rows + lead_rows
        pages = [-(-t // page) for t in kv_lens]
        self.n_pages = sum(pages) + spare
        order = rng.permutation(self.n_pages).astype(np.int32)
        self.max_pages = max(pages + [1])
        table = np.full((n, self.max_pages), -7, np.int32)
        at = 0
        for i, p in enumerate(pages):
            table[i, :p] = order[at:at + p]
            at += p
        self.table_host = table
        self.table = torch.from_numpy(table).cuda()
        self.q_start_host = lead_rows + np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
        self.q_start = torch.from_numpy(self.q_start_host.astype(np.int32)).cuda()
        self.kv_len = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
        shape = (self.n_pages, hkv, page, dim) if layout == "head" else (self.n_pages, page, hkv, dim)
        self.k = torch.full(shape, math.nan, dtype=self.t, device="cuda")
        self.v = torch.full(shape, math.nan, dtype=self.t, device="cuda")

    def desc(self, **kw):
        if self.layout == "token":
            kw = dict(head_stride=self.dim, token_stride=self.hkv * self.dim, **kw)
        kw.setdefault("max_q", max(self.q_lens + [0]))
        return P.PagedDesc(n_seq=len(self.q_lens), n_tokens=self.n_tokens, n_head_q=self.hq, n_head_kv=self.hkv,
                           page_size=self.page, n_pages=self.n_pages, max_pages=self.max_pages, head_dim=self.dim,
                           dtype=self.kind, **kw)

    def slots(self, s, lo=0):
        where = np.arange(lo, self.kv_lens[s])
        page = self.torch.from_numpy(self.table_host[s][where // self.page].astype(np.int64)).cuda()
        return page, self.torch.from_numpy(where % self.page).cuda()

    def rows(self, x, s, lo=0):
        """[tokens, n_head_kv, dim] of sequence s in pages x, in 64 bits."""
        page, off = self.slots(s, lo)
        return (x[page, :, off] if self.layout == "head" else x[page, off]).double()

    def fill(self, scale=1.0):
        torch = self.torch
        for s in range(len(self.q_lens)):
            page, off = self.slots(s)
            for x in (self.k, self.v):
                r = (torch.randn(len(page), self.hkv, self.dim, generator=self.gen, device="cuda") * scale).to(self.t)
                if self.layout == "head":
                    x[page, :, off] = r
                else:
                    x[page, off] = r

    def queries(self, scale=1.5):
        return (self.torch.randn(self.n_tokens, self.hq, self.dim, generator=self.gen, device="cuda") * scale).to(self.t)


def attend64(b, q, scale=0.0, softcap=0.0, causal=True):
    """(o, lse, bound of o, bound of lse) in 64 bits; rows of no sequence stay NaN."""
    torch = b.torch
    scale = scale or 1.0 / math.sqrt(b.dim)
    group = b.hq // b.hkv
    u = torch.finfo(b.t).eps / 2
    o = torch.full((b.n_tokens, b.hq, b.dim), math.nan, dtype=torch.float64, device="cuda")
    lse = torch.full((b.n_tokens, b.hq), math.nan, dtype=torch.float64, device="cuda")
    tol_o, tol_l = torch.zeros_like(o), torch.zeros_like(lse)
    for s, (n, t) in enumerate(zip(b.q_lens, b.kv_lens)):
        if n == 0:
            continue
        lo = int(b.q_start_host[s])
        k, v = b.rows(b.k, s), b.rows(b.v, s)
        for h in range(b.hq):
            qh, kh, vh = q[lo:lo + n, h].double(), k[:, h // group], v[:, h // group]
            x = qh @ kh.T * scale
            err = b.dim * 2.0 ** -24 * abs(scale) * (qh.abs() @ kh.abs().T) + 2.0 ** -20
            if softcap:
                x = torch.tanh(x / softcap) * softcap
                err = err + 2.0 ** -20 * softcap
            if causal:
                seen = torch.arange(t, device="cuda")[None] < (t - n + 1 + torch.arange(n, device="cuda"))[:, None]
                x = torch.where(seen, x, torch.full_like(x, -math.inf))
                err = torch.where(seen, err, torch.zeros_like(err))
            if t == 0:
                o[lo:lo + n, h], lse[lo:lo + n, h] = 0.0, -math.inf
                continue
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


def check(torch, b, o, lse, want):
    ro, rl, to, tl = want
    rows = ~torch.isnan(rl)
    empty = torch.isneginf(rl)
    assert torch.equal(torch.isneginf(lse) & rows, empty), "rows that see no key"
    assert bool((o[empty].float() == 0).all())
    live = rows & ~empty
    d = (o.double() - ro).abs()[live]
    assert bool((d <= to[live]).all()), f"o off by {float((d / to[live]).max()):.3g} of the bound"
    d = (lse.double() - rl).abs()[live]
    assert bool((d <= tl[live]).all()), f"lse off by {float((d / tl[live]).max()):.3g} of the bound"


def attend(b, q, **kw):
    d = b.desc(**kw)
    o, lse = P.fa_paged(d, q, b.k, b.v, b.table, b.q_start, b.kv_len)
    P.check(P.device_error())
    return o, lse


# lengths of one, around a tile and a page, several sequences
CASES = [
    # q_lens, kv_lens, hq, hkv, dim, dtype, page, layout
    ([1], [1], 1, 1, 64, "f16", 1, "head"),
    ([1], [4096], 32, 8, 128, "f16", 16, "head"),
    ([1, 1, 1], [63, 64, 65], 4, 2, 128, "bf16", 7, "token"),
    ([1] * 9, [1, 2, 127, 128, 129, 1000, 3, 511, 77], 8, 1, 64, "bf16", 24, "head"),
    ([2, 5, 1], [2, 300, 1], 6, 2, 128, "f16", 33, "token"),
    ([1], [2500], 24, 1, 128, "f16", 64, "head"),          # more query heads than a row tile of 16
    ([100], [100], 4, 4, 64, "f16", 16, "head"),
    ([129, 1, 64], [129, 700, 64], 8, 2, 128, "bf16", 32, "token"),
    ([300], [1333], 10, 2, 128, "f16", 128, "head"),        # 5 heads of a group: rows off the token grid
    ([257, 31], [257, 2000], 3, 1, 64, "bf16", 256, "head"),
    ([77], [513], 14, 2, 128, "f16", 9, "head"),            # pages of 9 tokens end inside every tile
    ([40, 200], [1000, 200], 8, 8, 128, "bf16", 8, "token"),
    ([700, 1, 1, 130], [900, 5, 2049, 4000], 16, 2, 64, "f16", 48, "head"),
    ([17 + i for i in range(20)], [60 + 11 * i for i in range(20)], 40, 40, 64, "f16", 16, "head"),   # 800 row tiles
    ([3000], [3500], 16, 16, 64, "bf16", 64, "token"),      # 192 row tiles of one sequence, several a CTA
    ([600, 555], [600, 1200], 144, 48, 64, "f16", 32, "head"),   # 672 row tiles, three query heads of a group
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(cuda, case, causal):
    q_lens, kv_lens, hq, hkv, dim, dtype, page, layout = CASES[case]
    b = Batch(cuda, q_lens, kv_lens, hq, hkv, dim, dtype, page, layout, seed=case)
    b.fill()
    q = b.queries()
    check(cuda, b, *attend(b, q, causal=causal), attend64(b, q, causal=causal))


@pytest.mark.parametrize("q_lens,kv_lens,page", [([1, 1], [400, 33], 16), ([150, 3], [400, 33], 16), ([150], [301], 5)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_softcap_scale_and_fp32_output(cuda, q_lens, kv_lens, page, dtype):
    b = Batch(cuda, q_lens, kv_lens, 8, 2, 128, dtype, page, seed=3)
    b.fill()
    q = b.queries(4.0)
    kw = dict(softcap=20.0, scale=0.2)
    check(cuda, b, *attend(b, q, **kw), attend64(b, q, **kw))
    o, lse = attend(b, q, o_fp32=True, **kw)
    assert o.dtype == cuda.float32
    check(cuda, b, o, lse, attend64(b, q, **kw))
    for kw in (dict(scale=-0.15), dict(scale=-0.15, softcap=20.0)):
        check(cuda, b, *attend(b, q, **kw), attend64(b, q, **kw))


@pytest.mark.parametrize("softcap", [1e-6, 1e-3, 0.5, 5.0, 100.0, 2000.0, 1e6])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [700, 5, 0]), ([300, 1, 40], [900, 3, 20])])
def test_caps_of_any_size(cuda, q_lens, kv_lens, softcap):
    """Caps below, among and far above the scores, rows without a key.  The bound allows the cap's rounding 2^-20 of it,
    except for the largest: cap tanh(x / cap) then differs from x by x^3 / (3 cap^2) < 1e-8, and no more is allowed."""
    b = Batch(cuda, q_lens, kv_lens, 6, 2, 64, "bf16", 16)
    b.fill()
    q = b.queries(2.0)
    for scale in (0.0, -0.2):
        o, lse = attend(b, q, softcap=softcap, scale=scale, causal=True, o_fp32=True)
        check(cuda, b, o, lse, attend64(b, q, scale, softcap if softcap < 1e6 else 0.0, True))


@pytest.mark.parametrize("rows", [1, 130])
def test_large_scores_and_rising_maxima(cuda, rows):
    """Scores whose maximum rises from tile to tile by far more than a rounding, and rows that one key decides."""
    b = Batch(cuda, [rows], [1000 + rows], 4, 1, 128, "f16", 16, seed=5)
    b.fill()
    page, off = b.slots(0)
    ramp = cuda.linspace(0.0, 6.0, len(page), device="cuda")[:, None, None]
    b.k[page, :, off] = (b.k[page, :, off].float() * ramp).to(b.t)
    q = b.queries(3.0)
    check(cuda, b, *attend(b, q), attend64(b, q))


@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("long", [False, True])
def test_empty_rows_and_padding(cuda, page, long):
    """Sequences without new tokens, without any token, more new tokens than keys; rows of no sequence are left."""
    q_lens, kv_lens = ([3, 0, 2, 1], [5, 7, 0, 64]) if not long else ([200, 0, 150, 1, 20], [300, 7, 0, 64, 11])
    b = Batch(cuda, q_lens, kv_lens, 4, 2, 64, "f16", page, seed=6, pad_rows=3, lead_rows=2)
    b.fill()
    q = b.queries()
    o = cuda.full((b.n_tokens, b.hq, b.dim), 7.0, dtype=b.t, device="cuda")
    lse = cuda.full((b.n_tokens, b.hq), 7.0, device="cuda")
    P.fa_paged(b.desc(), q, b.k, b.v, b.table, b.q_start, b.kv_len, o=o, lse=lse)
    P.check(P.device_error())
    outside = cuda.ones(b.n_tokens, dtype=cuda.bool, device="cuda")
    outside[2:2 + sum(q_lens)] = False
    assert bool((o[outside] == 7).all()) and bool((lse[outside] == 7).all())
    want = attend64(b, q)
    check(cuda, b, o[:], lse, want)


@pytest.mark.parametrize("q_lens,kv_lens,page", [([1, 1, 1], [500, 20, 129], 16), ([140, 1], [500, 129], 16)])
def test_strided_rows(cuda, q_lens, kv_lens, page):
    """q as a slice of a fused row, o with a gap behind every row, pages inside larger ones."""
    b = Batch(cuda, q_lens, kv_lens, 8, 2, 64, "bf16", page, seed=8)
    b.fill()
    n, w = b.n_tokens, b.hq * b.dim
    fused = cuda.full((n, w + 128), math.nan, dtype=b.t, device="cuda")
    q = b.queries()
    fused[:, :w] = q.view(n, w)
    wide_k = cuda.full((b.n_pages, 2, b.hkv, b.page, b.dim), math.nan, dtype=b.t, device="cuda")
    wide_k[:, 0], wide_k[:, 1] = b.k, b.v
    out = cuda.full((n, w + 8), 7.0, dtype=b.t, device="cuda")
    d = b.desc(q_stride=w + 128, o_stride=w + 8, page_stride=2 * b.hkv * b.page * b.dim)
    lse = cuda.empty(n, b.hq, device="cuda")
    P.fa_paged(d, fused[:, :w], wide_k, wide_k[:, 1], b.table, b.q_start, b.kv_len, o=out[:, :w], lse=lse)
    P.check(P.device_error())
    assert bool((out[:, w:] == 7).all())
    check(cuda, b, out[:, :w].reshape(n, b.hq, b.dim), lse, attend64(b, q))


def test_agrees_with_the_contiguous_decode(cuda):
    """One token over pages against p100_fa_decode over the same rows in one piece."""
    b = Batch(cuda, [1], [777], 8, 2, 128, "f16", 16, seed=9)
    b.fill()
    q = b.queries()
    o, lse = attend(b, q, o_fp32=True)
    k, v = (b.rows(x, 0).half().permute(1, 0, 2).contiguous() for x in (b.k, b.v))
    d = P.AttnDesc(n_head_q=8, n_head_kv=2, seq_kv=777)
    o2, lse2 = P.fa_decode(d, q.float().view(1, 8, 1, 128), k, v)
    _, _, tol, tol_l = attend64(b, q)
    assert bool(((o - o2.view(1, 8, 128)).abs() <= 2 * tol).all())
    assert bool(((lse - lse2.view(1, 8)).abs() <= 2 * tol_l).all())


@pytest.mark.parametrize("q_lens,page", [([1, 1, 1, 1], 16), ([70, 1, 300, 9], 16), ([70, 1], 7)])
def test_same_bits_again_in_a_graph_on_another_stream(cuda, q_lens, page):
    """A captured call follows new lengths and tables; repeated calls give the same bits; a shared workspace."""
    torch = cuda
    kv = [900 + 37 * i for i in range(len(q_lens))]
    b = Batch(torch, q_lens, kv, 8, 2, 128, "f16", page, seed=10)
    b.fill()
    q = b.queries()
    d = b.desc()
    ws = P.fa_paged_workspace(d)
    o, lse = P.fa_paged(d, q, b.k, b.v, b.table, b.q_start, b.kv_len, ws=ws)
    first = (o.clone(), lse.clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    o2, lse2 = P.fa_paged(d, q, b.k, b.v, b.table, b.q_start, b.kv_len, stream=side)
    side.synchronize()
    assert torch.equal(o2, first[0]) and torch.equal(lse2, first[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        P.fa_paged(d, q, b.k, b.v, b.table, b.q_start, b.kv_len, o=o, lse=lse, ws=ws)
    for _ in range(3):
        o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, first[0]) and torch.equal(lse, first[1])
    # fewer keys: the graph reads the lengths when it runs
    b.kv_lens = [max(n, t // 3) for n, t in zip(q_lens, kv)]
    b.kv_len.copy_(torch.tensor(b.kv_lens, dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    check(torch, b, o, lse, attend64(b, q))
    P.check(P.device_error())


@pytest.mark.parametrize("q_lens,page", [([1, 1], 16), ([90, 1], 16), ([90, 1], 3)])
def test_bad_lengths_and_pages_are_reported(cuda, q_lens, page):
    """Nothing is written for lengths out of order; a page out of range is not read; both raise the flag."""
    torch = cuda
    b = Batch(torch, q_lens, [300, 40], 4, 1, 64, "f16", page, seed=11)
    b.fill()
    q = b.queries()
    o = torch.full((b.n_tokens, b.hq, b.dim), 7.0, dtype=b.t, device="cuda")
    n = q_lens[0]
    for starts, lens in (([0, n, n - 1], [300, 40]), ([0, n, n + 1], [-1, 40]), ([0, n, n + 2], [300, 40]),
                         ([-1, n, n + 1], [300, 40]), ([0, n, n + 1], [300, b.max_pages * page + 1])):
        P.fa_paged(b.desc(), q, b.k, b.v, b.table, torch.tensor(starts, dtype=torch.int32, device="cuda"),
                   torch.tensor(lens, dtype=torch.int32, device="cuda"), o=o)
        with pytest.raises(P.InvalidArgument):
            P.check(P.device_error())
        assert bool((o == 7).all())
    table = b.table.clone()
    table[0, 1], table[1, 0] = b.n_pages, -1
    P.fa_paged(b.desc(), q, b.k, b.v, table, b.q_start, b.kv_len, o=o)
    with pytest.raises(P.InvalidArgument):
        P.check(P.device_error())
    o, lse = attend(b, q)   # and the next call is clean
    check(torch, b, o, lse, attend64(b, q))


@pytest.mark.parametrize("n,long", [(130, 1), (300, 20), (1024, 1), (1024, 18)])
def test_many_sequences(cuda, n, long):
    """More sequences than a block has threads, up to the largest batch."""
    rng = np.random.RandomState(n)
    q_lens = [int(x) for x in rng.randint(0, long + 1, n)]
    q_lens[-1] = long
    kv_lens = [int(q + rng.randint(0, 90)) for q in q_lens]
    b = Batch(cuda, q_lens, kv_lens, 2, 1, 64, "f16", 16, seed=n)
    b.fill()
    q = b.queries()
    check(cuda, b, *attend(b, q), attend64(b, q))


@pytest.mark.parametrize("q_len,page", [(1, 16), (40, 16), (40, 6)])
def test_offsets_beyond_32_bits(cuda, q_len, page):
    """Pages 3 GB apart: the last one starts 6 billion elements behind the first."""
    torch = cuda
    n_pages, hkv, dim, gap = 5, 2, 64, 1_500_000_000 // 8 * 8
    kv = n_pages * page - 3
    store = torch.empty((n_pages - 1) * gap + hkv * page * dim, dtype=torch.float16, device="cuda")
    b = Batch(torch, [q_len], [kv if kv > q_len else q_len], 4, hkv, dim, "f16", page, seed=50, spare=0)
    n_pages = b.n_pages
    shape, strides = (n_pages, hkv, page, dim), (gap, page * dim, dim, 1)
    if (n_pages - 1) * gap + hkv * page * dim > store.numel():
        store = torch.empty((n_pages - 1) * gap + hkv * page * dim, dtype=torch.float16, device="cuda")
    b.k = store.as_strided(shape, strides)
    b.v = torch.empty_like(store).as_strided(shape, strides)
    b.k.fill_(math.nan)
    b.v.fill_(math.nan)
    first = b.kv_lens[0] - q_len
    b.fill()
    qkv = torch.randn(q_len, (4 + 2 * hkv) * dim, generator=b.gen, device="cuda")
    d = b.desc(page_stride=gap)
    q = P.paged_append(d, qkv, b.table, b.q_start, b.kv_len, b.k, b.v)
    want, length, ks = append64(b, qkv, None, None, None, 0.0, False)
    near(torch, b.t, q, want, length)
    near(torch, b.t, b.rows(b.k, 0, first), ks[0][0], ks[0][1])
    o, lse = P.fa_paged(d, q, b.k, b.v, b.table, b.q_start, b.kv_len)
    P.check(P.device_error())
    check(torch, b, o, lse, attend64(b, q))


@pytest.mark.parametrize("q_lens", [[1, 1, 1], [60, 200, 1]])
def test_sequences_that_share_pages(cuda, q_lens):
    """A common prefix held once: three block tables begin with the same pages."""
    b = Batch(cuda, q_lens, [100 + 64 + n for n in q_lens], 8, 2, 128, "bf16", 32, seed=51)
    for i in (1, 2):
        b.table_host[i, :4] = b.table_host[0, :4]
    b.table.copy_(cuda.from_numpy(b.table_host))
    b.fill()
    q = b.queries()
    check(cuda, b, *attend(b, q), attend64(b, q))


@pytest.mark.parametrize("q_lens", [[1, 1], [300, 1]])
def test_two_calls_at_once_and_no_lse(cuda, q_lens):
    """Two streams with a workspace each; lse left out through the C interface."""
    import ctypes as C
    torch = cuda
    b = Batch(torch, q_lens, [3000, 2000], 16, 4, 128, "f16", 16, seed=52)
    b.fill()
    qs = [b.queries() for _ in range(2)]
    d = b.desc()
    want = [P.fa_paged(d, q, b.k, b.v, b.table, b.q_start, b.kv_len)[0].clone() for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    spaces = [P.fa_paged_workspace(d) for _ in range(2)]
    outs = [torch.empty_like(w) for w in want]
    torch.cuda.synchronize()
    for _ in range(20):
        for q, st, ws, o in zip(qs, streams, spaces, outs):
            P.check(P.lib().p100_fa_paged(C.byref(d), q.data_ptr(), b.k.data_ptr(), b.v.data_ptr(), b.table.data_ptr(),
                                          b.q_start.data_ptr(), b.kv_len.data_ptr(), o.data_ptr(), None, ws.data_ptr(),
                                          ws.numel(), st.cuda_stream))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    P.check(P.device_error())


# ------------------------------------------------------------------ append
def append64(b, qkv, rope, q_norm, k_norm, eps, half):
    """(q [n_tokens, hq, dim], k and v per sequence, the pairs' lengths of q and k) in 64 bits."""
    torch = b.torch
    out = torch.full((b.n_tokens, b.hq, b.dim), math.nan, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    ks = []
    for s, (n, t) in enumerate(zip(b.q_lens, b.kv_lens)):
        lo = int(b.q_start_host[s])
        x = qkv[lo:lo + n].double().view(n, b.hq + 2 * b.hkv, b.dim)
        parts = [x[:, :b.hq], x[:, b.hq:b.hq + b.hkv]]
        mags = []
        for i, w in enumerate((q_norm, k_norm)):
            if w is not None:
                parts[i] = parts[i] / torch.sqrt(parts[i].square().mean(-1, keepdim=True) + eps) * w.double()
            if rope is not None:
                cs = rope[t - n:t].double()[:, None]
                h = b.dim // 2
                a, c = (parts[i][..., :h], parts[i][..., h:]) if half else (parts[i][..., 0::2], parts[i][..., 1::2])
                y = (a * cs[..., 0] - c * cs[..., 1], a * cs[..., 1] + c * cs[..., 0])
                length = torch.sqrt(a * a + c * c)
                parts[i] = torch.cat(y, -1) if half else torch.stack(y, -1).flatten(-2)
                mags.append(torch.cat((length, length), -1) if half else torch.stack((length, length), -1).flatten(-2))
            else:
                mags.append(parts[i].abs())
        out[lo:lo + n], mag[lo:lo + n] = parts[0], mags[0]
        ks.append((parts[1], mags[1], x[:, b.hq + b.hkv:]))
    return out, mag, ks


def near(torch, t, got, want, length):
    u = torch.finfo(t).eps / 2
    tol = u * want.abs() + (1 + u) * 2.0 ** -18 * length + torch.finfo(t).tiny * torch.finfo(t).eps
    d = (got.double() - want).abs()
    assert bool((d <= tol).all()), f"off by {float((d / tol).max()):.3g} of the bound"


APPENDS = [
    # q_lens, kv_lens, hq, hkv, dim, src, dtype, page, layout, norm, rope, half
    ([1], [1], 1, 1, 64, "f32", "f16", 1, "head", False, True, False),
    ([1], [4096], 32, 8, 128, "f32", "f16", 16, "head", False, True, False),
    ([5, 1, 33], [70, 1, 33], 6, 2, 128, "bf16", "bf16", 7, "token", True, True, True),
    ([100, 0, 40], [163, 9, 1000], 8, 1, 64, "f16", "f16", 24, "head", True, True, False),
    ([17], [40], 5, 5, 64, "f32", "bf16", 64, "token", True, False, False),
    ([64, 3], [64, 130], 3, 1, 128, "f16", "bf16", 32, "head", False, True, True),
    ([2] * 70, [3 + i for i in range(70)], 4, 2, 64, "bf16", "f16", 16, "head", False, False, False),
]


@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(cuda, case):
    torch = cuda
    q_lens, kv_lens, hq, hkv, dim, src, dtype, page, layout, norm, rope, half = APPENDS[case]
    b = Batch(torch, q_lens, kv_lens, hq, hkv, dim, dtype, page, layout, seed=20 + case, pad_rows=2, lead_rows=1)
    qkv = (torch.randn(b.n_tokens, (hq + 2 * hkv) * dim, generator=b.gen, device="cuda") * 2).to(types(torch)[src][0])
    table = torch.from_numpy(P.rope_table(max(kv_lens), dim, 10000.0)).cuda() if rope else None
    w = [torch.rand(dim, generator=b.gen, device="cuda") + 0.5 if norm else None for _ in range(2)]
    q = torch.full((b.n_tokens, hq, dim), 7.0, dtype=b.t, device="cuda")
    d = b.desc()
    P.paged_append(d, qkv, b.table, b.q_start, b.kv_len, b.k, b.v, rope_cs=table, q_norm=w[0], k_norm=w[1], eps=1e-6,
                   rope_half=half, q=q)
    P.check(P.device_error())
    want, length, ks = append64(b, qkv, table, w[0], w[1], 1e-6, half)
    rows = ~torch.isnan(want)
    assert bool((q[~rows] == 7).all())
    near(torch, b.t, q[rows], want[rows], length[rows])
    written = 0
    for s, (k, klen, v) in enumerate(ks):
        first = kv_lens[s] - q_lens[s]
        near(torch, b.t, b.rows(b.k, s, first), k, klen)
        near(torch, b.t, b.rows(b.v, s, first), v, v.abs() * 0)
        written += k.numel()
    for x in (b.k, b.v):   # every other row of the pages is as it was
        assert int((~torch.isnan(x)).sum()) == written


def test_append_reports_bad_positions(cuda):
    torch = cuda
    b = Batch(torch, [4, 4], [4, 10], 2, 1, 64, "f16", 4, seed=30)
    qkv = torch.randn(8, 4 * 64, device="cuda")
    rope = torch.from_numpy(P.rope_table(8, 64, 10000.0)).cuda()   # positions 8, 9 are missing
    q = torch.full((8, 2, 64), 7.0, dtype=b.t, device="cuda")
    P.paged_append(b.desc(), qkv, b.table, b.q_start, b.kv_len, b.k, b.v, rope_cs=rope, q=q)
    with pytest.raises(P.InvalidArgument):
        P.check(P.device_error())
    assert bool((q[6:] == 7).all()) and not bool((q[:6] == 7).any())
    assert int((~torch.isnan(b.k)).sum()) == 6 * 64
    for table, kv in ((torch.full_like(b.table, b.n_pages), [4, 8]), (b.table, [3, 8])):
        k = torch.full_like(b.k, math.nan)
        P.paged_append(b.desc(), qkv, table, b.q_start, torch.tensor(kv, dtype=torch.int32, device="cuda"), k,
                       b.v.clone(), rope_cs=rope)
        with pytest.raises(P.InvalidArgument):
            P.check(P.device_error())
    P.paged_append(b.desc(), qkv, b.table, b.q_start, b.kv_len, b.k, b.v)
    P.check(P.device_error())


def test_append_strided_rows_and_graph(cuda):
    torch = cuda
    b = Batch(torch, [3, 6], [20, 6], 4, 2, 64, "f16", 8, seed=31)
    wide = torch.randn(9, 8 * 64 + 16, generator=b.gen, device="cuda")
    qkv = wide[:, :8 * 64]
    d = b.desc(q_stride=4 * 64 + 8)
    rope = torch.from_numpy(P.rope_table(20, 64, 10000.0)).cuda()
    q = torch.full((9, 4 * 64 + 8), 7.0, dtype=b.t, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        P.paged_append(d, qkv, b.table, b.q_start, b.kv_len, b.k, b.v, rope_cs=rope, q=q[:, :256])
    graph.replay()
    torch.cuda.synchronize()
    P.check(P.device_error())
    want, length, ks = append64(b, qkv, rope, None, None, 0.0, False)
    near(torch, b.t, q[:, :256].reshape(9, 4, 64), want, length)
    assert bool((q[:, 256:] == 7).all())
    near(torch, b.t, b.rows(b.k, 0, 17), ks[0][0], ks[0][1])


def test_prompt_in_chunks_then_tokens(cuda):
    """Two sequences served together: a prompt in one piece and in chunks, then single tokens, through append,
    attention and the scoring of logits; every stage against 64 bits on the device's own inputs."""
    torch = cuda
    hq, hkv, dim, page, vocab = 8, 2, 64, 16, 517
    width = (hq + 2 * hkv) * dim
    gen = torch.Generator(device="cuda")
    gen.manual_seed(40)
    total = [150, 83]
    rows = [torch.randn(t, width, generator=gen, device="cuda") for t in total]
    rope = torch.from_numpy(P.rope_table(160, dim, 10000.0)).cuda()
    norm = torch.rand(dim, generator=gen, device="cuda") + 0.5
    head = torch.randn(hq * dim, vocab, generator=gen, device="cuda")
    full = Batch(torch, total, total, hq, hkv, dim, "f16", page, seed=41)
    steps = [([70, 0], [70, 0]), ([79, 80], [149, 80])] + [([1 if i == 0 else 0, 1], [150, 81 + i]) for i in range(3)]

    def step(b, qkv):
        q = P.paged_append(b.desc(), qkv, b.table, b.q_start, b.kv_len, b.k, b.v, rope_cs=rope, q_norm=norm,
                           k_norm=norm, eps=1e-6)
        o, lse = P.fa_paged(b.desc(o_fp32=True), q, b.k, b.v, b.table, b.q_start, b.kv_len)
        check(torch, b, o, lse, attend64(b, q))
        return q, o

    q_full, o_full = step(full, torch.cat(rows))
    logits = (o_full.view(sum(total), -1) @ head)
    tokens = torch.randint(0, vocab, (sum(total),), generator=gen, device="cuda", dtype=torch.int32)
    r = P.logprobs(logits, tokens, top_k=3)
    y = torch.log_softmax(logits.double(), 1)
    assert torch.allclose(r.logprob.double(), y.gather(1, tokens.long()[:, None])[:, 0], rtol=1e-5, atol=1e-5)
    assert torch.equal(r.top_index[:, 0].long(), logits.argmax(1))

    b = Batch(torch, total, total, hq, hkv, dim, "f16", page, seed=42)
    got = [[], []]
    for q_lens, kv_lens in steps:
        b.q_lens, b.kv_lens, b.n_tokens = q_lens, kv_lens, sum(q_lens)
        b.q_start_host = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
        b.q_start = torch.from_numpy(b.q_start_host).cuda()
        b.kv_len = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
        qkv = torch.cat([rows[s][kv_lens[s] - q_lens[s]:kv_lens[s]] for s in range(2)])
        q, o = step(b, qkv)
        for s in range(2):
            got[s].append((q[b.q_start_host[s]:b.q_start_host[s + 1]], o[b.q_start_host[s]:b.q_start_host[s + 1]]))
    for s in range(2):   # the same cache and queries, bit for bit; the outputs within both calls' bounds
        lo = int(full.q_start_host[s])
        assert torch.equal(torch.cat([x[0] for x in got[s]]), q_full[lo:lo + total[s]])
        assert torch.equal(b.rows(b.k, s), full.rows(full.k, s)) and torch.equal(b.rows(b.v, s), full.rows(full.v, s))
    tol = attend64(full, q_full)[2]
    for s in range(2):
        lo = int(full.q_start_host[s])
        d = (torch.cat([x[1] for x in got[s]]) - o_full[lo:lo + total[s]]).abs()
        assert bool((d <= 2 * tol[lo:lo + total[s]]).all())
