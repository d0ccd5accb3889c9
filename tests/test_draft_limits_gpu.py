"""Calls for steps and drafted trees at their limits: far pages, strided rows, unseen rows that hold NaN, graphs that
follow new trees beside a second call, two calls at once, the largest trees.  Tolerances as in test_draft_gpu."""
import ctypes as C
import math

import numpy as np
import pytest

import p100_b200 as P
from test_draft_gpu import append64, attend_tree, mask_of, masks, random_tree, tree64
from test_paged_gpu import Batch, check, near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_len,page", [(2, 16), (40, 16), (40, 6)])
def test_offsets_beyond_32_bits(cuda, q_len, page):
    """Pages 3 GB apart: the last one starts 6 billion elements behind the first."""
    torch = cuda
    hkv, dim, gap = 2, 64, 1_500_000_000 // 8 * 8
    b = Batch(torch, [q_len], [max(5 * page - 3, q_len)], 4, hkv, dim, "f16", page, seed=50, spare=0)
    store = torch.empty((b.n_pages - 1) * gap + hkv * page * dim, dtype=torch.float16, device="cuda")
    shape, strides = (b.n_pages, hkv, page, dim), (gap, page * dim, dim, 1)
    b.k = store.as_strided(shape, strides)
    b.v = torch.empty_like(store).as_strided(shape, strides)
    b.k.fill_(math.nan)
    b.v.fill_(math.nan)
    b.fill()
    first = b.kv_lens[0] - q_len
    qkv = torch.randn(q_len, (4 + 2 * hkv) * dim, generator=b.gen, device="cuda")
    d = b.desc(page_stride=gap)
    where = (b.table, b.q_start, b.kv_len)
    kw = dict(rope_dim=32, theta=10000.0)
    q = P.paged_append_rope(d, qkv, P.Rope(**kw), *where, b.k, b.v)
    (want, length), (k, klen), v = append64(b, qkv, kw, False, np.arange(first, first + q_len), None, None, 0.0)
    near(torch, b.t, q, want, length)
    near(torch, b.t, b.rows(b.k, 0, first), k, klen)
    mask, bits = masks(b, np.random.RandomState(0), "any", 2)
    o, lse = P.fa_tree(d, q, b.k, b.v, mask, *where)
    P.check(P.device_error())
    check(torch, b, o, lse, tree64(b, q, bits))
    rows = [b.rows(x, 0, first).clone() for x in (b.k, b.v)]
    keep = torch.zeros(q_len, dtype=torch.int32, device="cuda")
    keep[0] = q_len - 1
    P.paged_keep(d, b.k, b.v, keep, torch.ones(1, dtype=torch.int32, device="cuda"), *where)
    P.check(P.device_error())
    for x, old in zip((b.k, b.v), rows):
        new = b.rows(x, 0, first)
        assert torch.equal(new[0], old[-1]) and torch.equal(new[1:], old[1:])


@pytest.mark.parametrize("q_lens,kv_lens,page", [([2, 1, 2], [500, 20, 129], 16), ([40, 9], [500, 129], 16)])
def test_strided_rows(cuda, q_lens, kv_lens, page):
    """q as a slice of a fused row, o with a gap behind every row, pages inside larger ones."""
    b = Batch(cuda, q_lens, kv_lens, 8, 2, 64, "bf16", page, seed=8)
    b.fill()
    n, w = b.n_tokens, b.hq * b.dim
    fused = cuda.full((n, w + 128), math.nan, dtype=b.t, device="cuda")
    q = b.queries()
    fused[:, :w] = q.view(n, w)
    wide = cuda.full((b.n_pages, 2, b.hkv, b.page, b.dim), math.nan, dtype=b.t, device="cuda")
    wide[:, 0], wide[:, 1] = b.k, b.v
    out = cuda.full((n, w + 8), 7.0, dtype=b.t, device="cuda")
    d = b.desc(q_stride=w + 128, o_stride=w + 8, page_stride=2 * b.hkv * b.page * b.dim)
    lse = cuda.empty(n, b.hq, device="cuda")
    mask, bits = masks(b, np.random.RandomState(0), "any", 2)
    P.fa_tree(d, fused[:, :w], wide, wide[:, 1], mask, b.table, b.q_start, b.kv_len, o=out[:, :w], lse=lse)
    P.check(P.device_error())
    assert bool((out[:, w:] == 7).all())
    check(cuda, b, out[:, :w].reshape(n, b.hq, b.dim), lse, tree64(b, q, bits))


@pytest.mark.parametrize("q_lens,kv_lens", [([6, 3], [300, 40]), ([50, 20], [300, 20])])
def test_hidden_keys_that_are_not_finite(cuda, q_lens, kv_lens):
    """Keys of tokens that no row of the tree sees may be NaN or infinite (their values have to be finite)."""
    torch = cuda
    for bad in (math.nan, math.inf, -math.inf):
        b = Batch(torch, q_lens, kv_lens, 4, 2, 64, "f16", 16, seed=4)
        b.fill()
        q = b.queries()
        mask, bits = masks(b, np.random.RandomState(0), "any", 2)
        bits = bits.clone()
        for s, n in enumerate(q_lens):   # nobody sees token n - 1, not even itself
            lo = int(b.q_start_host[s])
            bits[lo:lo + n, n - 1] = False
        packed = np.packbits(bits.cpu().numpy(), axis=1, bitorder="little").view(np.int32)
        mask = torch.from_numpy(packed).cuda()
        clean = b.k.clone()
        for s in range(len(q_lens)):
            page, off = b.slots(s, kv_lens[s] - 1)
            b.k[page, :, off] = bad
            clean[page, :, off] = 0
        o, lse = attend_tree(b, q, mask)
        b.k = clean
        check(torch, b, o, lse, tree64(b, q, bits))


@pytest.mark.parametrize("sizes,page", [([3, 2, 4], 16), ([60, 8, 33], 16), ([60, 8], 7)])
def test_graph_follows_new_trees_beside_a_second_call(cuda, sizes, page):
    """A captured call with other lengths, tables and masks at each replay, another stream's call (a workspace of its own)
    at the same time; repeated replays give the same bits."""
    torch = cuda
    rng = np.random.RandomState(0)
    most = [n + 5 for n in sizes]
    b = Batch(torch, most, [900 + 37 * i + n for i, n in enumerate(most)], 8, 2, 128, "f16", page, seed=10)
    b.fill()
    other = Batch(torch, [30, 1], [2000, 700], 8, 2, 128, "f16", 16, seed=11)
    other.fill()
    oq, (om, obits) = other.queries(), masks(other, rng, "any", 1)
    want_other = tree64(other, oq, obits)
    q = b.queries()
    d, words = b.desc(), 3
    ws, ws2 = P.fa_paged_workspace(d), P.fa_paged_workspace(other.desc())
    mask = torch.zeros((b.n_tokens, words), dtype=torch.int32, device="cuda")
    o, lse = P.fa_tree(d, q, b.k, b.v, mask, b.table, b.q_start, b.kv_len, ws=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        P.fa_tree(d, q, b.k, b.v, mask, b.table, b.q_start, b.kv_len, o=o, lse=lse, ws=ws)
    side = torch.cuda.Stream()
    for step in range(4):
        b.q_lens = [max(1, n - step) for n in sizes]
        b.kv_lens = [n + int(rng.randint(0, 800)) for n in b.q_lens]
        b.q_start_host = np.concatenate([[0], np.cumsum(b.q_lens)]).astype(np.int32)
        b.q_start.copy_(torch.from_numpy(b.q_start_host))
        b.kv_len.copy_(torch.tensor(b.kv_lens, dtype=torch.int32))
        new, bits = masks(b, rng, "any", words)
        mask.copy_(new)
        torch.cuda.synchronize()
        got = []
        for _ in range(2):
            o.fill_(7.0)
            graph.replay()
            o2, lse2 = P.fa_tree(other.desc(), oq, other.k, other.v, om, other.table, other.q_start, other.kv_len, ws=ws2,
                                 stream=side)
            torch.cuda.synchronize()
            got.append((o.clone(), lse.clone()))
            check(torch, other, o2, lse2, want_other)
        assert torch.equal(got[0][0], got[1][0])
        end = int(b.q_start_host[-1])
        assert torch.equal(got[0][1][:end], got[1][1][:end]) and bool((o[end:] == 7).all())
        check(torch, b, o, lse, tree64(b, q, bits))
    P.check(P.device_error())


@pytest.mark.parametrize("q_lens", [[2, 1], [40, 3]])
def test_two_calls_at_once_and_no_lse(cuda, q_lens):
    torch = cuda
    b = Batch(torch, q_lens, [3000, 2000], 16, 4, 128, "f16", 16, seed=52)
    b.fill()
    qs = [b.queries() for _ in range(2)]
    d = b.desc()
    mask, _ = masks(b, np.random.RandomState(0), "any", 2)
    want = [P.fa_tree(d, q, b.k, b.v, mask, b.table, b.q_start, b.kv_len)[0].clone() for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    spaces = [P.fa_paged_workspace(d) for _ in range(2)]
    outs = [torch.empty_like(w) for w in want]
    torch.cuda.synchronize()
    for _ in range(20):
        for q, st, ws, o in zip(qs, streams, spaces, outs):
            P.check(P.lib().p100_fa_tree(C.byref(d), q.data_ptr(), b.k.data_ptr(), b.v.data_ptr(), mask.data_ptr(), 2,
                                         b.table.data_ptr(), b.q_start.data_ptr(), b.kv_len.data_ptr(), o.data_ptr(), None,
                                         ws.data_ptr(), ws.numel(), st.cuda_stream))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    P.check(P.device_error())


def test_one_workspace_for_trees_and_prompts(cuda):
    """Calls of both attentions that follow one another on one workspace, kernels of each kind."""
    torch = cuda
    batches = [Batch(torch, q, kv, 16, 4, 64, "bf16", 16, seed=60 + i) for i, (q, kv) in enumerate(
        (([1, 1, 1], [2500, 30, 700]), ([300, 1], [900, 4000]), ([4, 2], [3000, 90]), ([60, 12], [3000, 500])))]
    ws = P.fa_paged_workspace(batches[0].desc())
    rng = np.random.RandomState(0)
    want = []
    for b in batches:
        b.fill()
        b.q = b.queries()
        mask, bits = masks(b, rng, "any", 10)
        b.mask = mask
        want.append(tree64(b, b.q, bits))
    from test_paged_gpu import attend64
    causal = [attend64(b, b.q) for b in batches]
    for _ in range(2):
        for b, w, c in zip(batches, want, causal):
            where = (b.table, b.q_start, b.kv_len)
            check(torch, b, *P.fa_tree(b.desc(), b.q, b.k, b.v, b.mask, *where, ws=ws), w)
            check(torch, b, *P.fa_paged(b.desc(), b.q, b.k, b.v, *where, ws=ws), c)
    P.check(P.device_error())


def test_many_sequences_of_small_trees(cuda):
    """1024 sequences, most of them one token, some empty, some without a context: row tiles dealt out whole."""
    rng = np.random.RandomState(3)
    q_lens = [int(rng.choice([0, 1, 1, 2, 5])) for _ in range(1024)]
    kv_lens = [n + int(rng.choice([0, 1, 40, 200])) for n in q_lens]
    for dim, hq, hkv in ((64, 8, 1), (128, 16, 2)):
        b = Batch(cuda, q_lens, kv_lens, hq, hkv, dim, "bf16", 16, seed=7)
        b.fill()
        q = b.queries()
        mask, bits = masks(b, rng, "any", 1)
        check(cuda, b, *attend_tree(b, q, mask), tree64(b, q, bits))


def test_mask_words_beyond_the_tree(cuda):
    """The same trees with one word and with the most: the same bits out."""
    b = Batch(cuda, [9, 30], [500, 77], 4, 1, 128, "f16", 16)
    b.fill()
    q = b.queries()
    rng = np.random.RandomState(0)
    parents = [random_tree(rng, n, "any") for n in b.q_lens]
    outs = []
    for words in (1, 2, 32):
        mask = cuda.from_numpy(mask_of(parents, words)[0]).cuda()
        outs.append(attend_tree(b, q, mask))
    for o, lse in outs[1:]:
        assert cuda.equal(o, outs[0][0]) and cuda.equal(lse, outs[0][1])


@pytest.mark.parametrize("n_seq,n_tokens", [(1, 4096), (1, 4097), (3, 20000), (1024, 60000)])
def test_plan_of_prompts(cuda, n_seq, n_tokens):
    """Long prompts planned at once, by one CTA and by a cluster."""
    torch = cuda
    rng = np.random.RandomState(n_seq)
    page = 16
    share = np.diff(np.concatenate([[0], np.sort(rng.randint(0, n_tokens, n_seq - 1)), [n_tokens]])).astype(int)
    length = rng.randint(0, 50, n_seq)
    max_pages = int((share + length).max()) // page + 1
    d = P.PagedDesc(n_seq=n_seq, n_tokens=n_tokens, n_head_q=1, n_head_kv=1, page_size=page,
                    n_pages=int(((share + length + page - 1) // page).sum()) + 2, max_pages=max_pages)
    pool, held, table = P.paged_pool(d)
    i32 = dict(dtype=torch.int32, device="cuda")
    r = P.paged_plan(d, torch.tensor(length.tolist(), **i32), torch.tensor(share.tolist(), **i32), pool, held, table)
    P.check(P.device_error())
    pos = np.concatenate([np.arange(a, a + n) for a, n in zip(length, share)])
    seq = np.repeat(np.arange(n_seq), share)
    t = table.cpu().numpy()
    assert np.array_equal(r.position.cpu().numpy(), pos)
    assert np.array_equal(r.slot.cpu().numpy(), t[seq, pos // page].astype(np.int64) * page + pos % page)
    used = t[t >= 0]
    assert len(np.unique(used)) == len(used) == int(((share + length + page - 1) // page).sum())
    assert int(pool[0]) == 2 and held.tolist() == ((share + length + page - 1) // page).tolist()


def test_slots_beyond_32_bits(cuda):
    """Slots are 64-bit numbers: pages of 2^20 tokens."""
    torch = cuda
    d = P.PagedDesc(n_seq=1, n_tokens=2, n_head_q=1, n_head_kv=1, page_size=1 << 20, n_pages=5000, max_pages=2)
    pool, held, table = P.paged_pool(d)
    pool[2:] = pool[2:].flip(0).contiguous()   # the last page on top
    i32 = dict(dtype=torch.int32, device="cuda")
    r = P.paged_plan(d, torch.tensor([(1 << 20) - 1], **i32), torch.tensor([2], **i32), pool, held, table)
    P.check(P.device_error())
    assert r.slot.tolist() == [4999 * (1 << 20) + (1 << 20) - 1, 4998 * (1 << 20)]


def test_other_streams(cuda):
    """Every call on a stream of its own, behind the work that made its inputs there."""
    torch = cuda
    side = torch.cuda.Stream()
    b = Batch(torch, [6, 3], [60, 33], 4, 2, 64, "f16", 8, seed=1)
    b.fill()
    rng = np.random.RandomState(0)
    parents = [random_tree(rng, n, "any") for n in b.q_lens]
    words, depth = mask_of(parents, 1)
    bits = torch.from_numpy(np.unpackbits(words.view(np.uint8), axis=1, bitorder="little").astype(bool)).cuda()
    qkv = torch.randn(9, 8 * 64, generator=b.gen, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        parent = torch.tensor(np.concatenate(parents).tolist(), dtype=torch.int32, device="cuda")
        late = qkv * 2
    where = (b.table, b.q_start, b.kv_len)
    tree = P.tree_mask(parent, b.q_start, b.kv_len, 1, stream=side)
    q = P.paged_append_rope(b.desc(), late, P.Rope(64, 10000.0), *where, b.k, b.v, position=tree.position, stream=side)
    o, lse = P.fa_tree(b.desc(), q, b.k, b.v, tree.mask, *where, stream=side)
    side.synchronize()
    P.check(P.device_error())
    check(torch, b, o, lse, tree64(b, q, bits))
    keep = torch.tensor([1, 4, 5, 0, 0, 0, 2, 0, 0], dtype=torch.int32, device="cuda")
    before = [b.rows(b.k, s, t - n).clone() for s, (n, t) in enumerate(zip(b.q_lens, b.kv_lens))]
    torch.cuda.synchronize()
    length = P.paged_keep(b.desc(), b.k, b.v, keep, torch.tensor([3, 1], dtype=torch.int32, device="cuda"), *where, stream=side)
    side.synchronize()
    assert length.tolist() == [57, 31]
    after = [b.rows(b.k, s, t - n) for s, (n, t) in enumerate(zip(b.q_lens, b.kv_lens))]
    assert torch.equal(after[0][:3], before[0][[1, 4, 5]]) and torch.equal(after[0][3:], before[0][3:])
    assert torch.equal(after[1][0], before[1][2]) and torch.equal(after[1][1:], before[1][1:])


@pytest.mark.parametrize("softcap,scale", [(1e-22, 1e-22), (3e-30, -1e-30), (1e-16, 2e-16), (1e-14, 1e-14)])
@pytest.mark.parametrize("q_lens,kv_lens", [([2, 1], [300, 70]), ([60, 3], [300, 70])])
def test_tiny_caps_with_tiny_scales(cuda, q_lens, kv_lens, softcap, scale):
    """Every score is next to zero, so a row's visible keys weigh the same; hidden ones must not weigh anything."""
    b = Batch(cuda, q_lens, kv_lens, 6, 2, 64, "bf16", 16, seed=60)
    b.fill()
    mask, bits = masks(b, np.random.RandomState(0), "any", 2)
    for size in (1.5, 0.01):
        q = b.queries(size)
        o, lse = attend_tree(b, q, mask, softcap=softcap, scale=scale, o_fp32=True)
        check(cuda, b, o, lse, tree64(b, q, bits, scale, softcap))


@pytest.mark.parametrize("softcap", [1e-6, 1e-3, 0.5, 5.0, 100.0, 2000.0, 1e6])
@pytest.mark.parametrize("q_lens,kv_lens", [([2, 1, 1], [700, 5, 1]), ([60, 1, 40], [900, 3, 40])])
def test_caps_of_any_size(cuda, q_lens, kv_lens, softcap):
    """As test_paged_gpu's: caps below, among and far above the scores; the largest may differ from none by 1e-8."""
    b = Batch(cuda, q_lens, kv_lens, 6, 2, 64, "bf16", 16)
    b.fill()
    mask, bits = masks(b, np.random.RandomState(0), "any", 2)
    q = b.queries(2.0)
    for scale in (0.0, -0.2):
        o, lse = attend_tree(b, q, mask, softcap=softcap, scale=scale, o_fp32=True)
        check(cuda, b, o, lse, tree64(b, q, bits, scale, softcap if softcap < 1e6 else 0.0))


@pytest.mark.parametrize("rows", [3, 60])
def test_large_scores_and_rising_maxima(cuda, rows):
    """Scores whose maximum rises from tile to tile by far more than a rounding, and rows that one key decides."""
    for dtype in ("f16", "bf16"):
        b = Batch(cuda, [rows], [1000 + rows], 4, 1, 128, dtype, 16, seed=5)
        b.fill()
        page, off = b.slots(0)
        grow = cuda.linspace(0.2, 6.0, 1000 + rows, device="cuda")[:, None, None]
        k = b.k[page, :, off].float() * grow
        b.k[page, :, off] = k.to(b.t)
        q = b.queries(2.0)
        mask, bits = masks(b, np.random.RandomState(0), "any", 2)
        check(cuda, b, *attend_tree(b, q, mask), tree64(b, q, bits))


@pytest.mark.parametrize("page,pages", [(8176, 262657), (114808, 18705)])   # 2^31 - 16 and 2^31 - 8 places
@pytest.mark.parametrize("n", [1, 9])
def test_as_many_keys_as_a_length_holds(cuda, n, page, pages):
    """A sequence of almost 2^31 tokens whose table names one page over and over, as test_paged_limits_gpu's: its keys are
    zero and weigh the same (V = 1); the newest token's own key (V = 3) decides its row, and no other row's bit names
    it; what the page holds behind the last token would decide every row if it took part.

    Bound: every term before the join is a whole number below 2^24 (of a power of two); the join adds at most 296 parts
    with relative errors of 2^-24 each in o and in the sum, and the one division rounds: below 2^-14."""
    torch = cuda
    dim, group, kv = 64, 4, page * pages - 3
    last = (kv - 1) % page
    t = torch.float16
    k = torch.zeros((2, 1, page, dim), dtype=t, device="cuda")
    v = torch.ones((2, 1, page, dim), dtype=t, device="cuda")
    k[1, 0, last], v[1, 0, last] = 5.0, 3.0
    k[1, 0, last + 1:], v[1, 0, last + 1:] = 10.0, 100.0
    table = torch.zeros((1, pages), dtype=torch.int32, device="cuda")
    table[0, -1] = 1
    q = torch.ones((n, group, dim), dtype=t, device="cuda")
    d = P.PagedDesc(n_seq=1, n_tokens=n, n_head_q=group, n_head_kv=1, page_size=page, n_pages=2, max_pages=pages,
                    head_dim=dim, o_fp32=True)
    mask = torch.from_numpy(mask_of([np.arange(-1, n - 1)], 1)[0]).cuda()
    o, lse = P.fa_tree(d, q, k, v, mask, table, torch.tensor([0, n], dtype=torch.int32, device="cuda"),
                       torch.tensor([kv], dtype=torch.int32, device="cuda"))
    P.check(P.device_error())
    x = 5.0 * dim / math.sqrt(dim)   # the newest key's score; the others' weight is below 2^31 e^-40 < 2^-26 of its own
    seen = math.log(kv - n + 1)
    assert bool(((o[:-1] - 1.0).abs() <= 2.0 ** -14).all())
    assert bool(((o[-1] - 3.0).abs() <= 3 * 2.0 ** -14).all())
    assert bool(((lse[:-1] - seen).abs() <= 2.0 ** -14 + 2.0 ** -22 * seen).all())
    assert bool(((lse[-1] - x).abs() <= 2.0 ** -14 + 2.0 ** -22 * x).all())


@pytest.mark.parametrize("n_seq,n_tokens", [(3, 16), (300, 900), (1000, 9000)])
def test_plan_goes_on_from_its_own_lengths(cuda, n_seq, n_tokens):
    """kv_len in length's place, as a captured step of single tokens has it: a CTA, a large CTA, a cluster."""
    torch = cuda
    d = P.PagedDesc(n_seq=n_seq, n_tokens=n_tokens, n_head_q=1, n_head_kv=1, page_size=4, n_pages=n_seq * 6, max_pages=6)
    pool, held, table = P.paged_pool(d)
    length = torch.arange(n_seq, dtype=torch.int32, device="cuda") % 5
    n_new = (torch.arange(n_seq, dtype=torch.int32, device="cuda") % 7 != 0).int() * 2
    apart = P.paged_plan(d, length, n_new, pool, held, table)
    out = P.PagedPlan(*(torch.empty_like(x) for x in apart))
    start, want = length.clone(), length.clone()
    here = out._replace(kv_len=start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        P.paged_plan(d, start, n_new, pool, held, table, out=here)
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        P.check(P.device_error())
        first = (n_new.cumsum(0) - n_new).tolist()
        place = here.position.tolist()
        for s in range(0, n_seq, 37):
            n, at = int(n_new[s]), first[s]
            assert place[at:at + n] == [int(want[s]) + i for i in range(n)]
        want += n_new
        assert torch.equal(start, want) and held.tolist() == [-(-x // 4) for x in want.tolist()]
