"""Plan, masks, append, attention and keep as steps of one captured graph, each call held to 64 bits on what the call before
it left: no rounding that may fall the other way has to be allowed for, so a mask, table, length or row that is handed on
wrongly shows.  Bounds: append as test_draft_gpu's, attention test_paged_gpu's, everything else bit for bit."""
import numpy as np
import pytest

import p100_b200 as P
from test_draft_gpu import append64, mask_of, random_tree, tree64
from test_paged_gpu import Batch, check, near, types

pytestmark = pytest.mark.gpu


def outside(torch, o, want):
    """The share of values that leave the bound."""
    ro, _, to, _ = want
    rows = ~torch.isnan(ro)
    return float(((o.double() - ro).abs() > to)[rows].double().mean())


@pytest.mark.parametrize("hq,hkv,dim,dtype,page,layout,draft", [
    (8, 2, 64, "f16", 8, "head", 9), (16, 2, 128, "bf16", 8, "head", 9), (16, 2, 128, "bf16", 7, "token", 9),
    (8, 4, 128, "f16", 16, "token", 7), (4, 4, 64, "bf16", 16, "head", 40), (3, 1, 128, "bf16", 4, "head", 4)])
def test_each_call_of_a_step_on_what_the_last_one_left(cuda, hq, hkv, dim, dtype, page, layout, draft):
    torch = cuda
    n_seq, steps, words = 5, 6, 1 + draft // 32
    t, kind = types(torch)[dtype]
    i32 = dict(dtype=torch.int32, device="cuda")
    max_pages = -(-(steps + 1) * draft // page)
    b = Batch(torch, [1] * n_seq, [1] * n_seq, hq, hkv, dim, dtype, page, layout, seed=hq)
    b.n_tokens, b.n_pages, b.max_pages = n_seq * draft, n_seq * max_pages, max_pages
    shape = (b.n_pages, hkv, page, dim) if layout == "head" else (b.n_pages, page, hkv, dim)
    k, v = torch.zeros(shape, dtype=t, device="cuda"), torch.zeros(shape, dtype=t, device="cuda")
    d = b.desc(max_q=draft)
    pool, held, table = P.paged_pool(d)
    kw = dict(rope_dim=dim // 2, theta=10000.0, scaling=P.ROPE_LINEAR, factor=2.0)
    rope, ws = P.Rope(half=True, **kw), P.fa_paged_workspace(d)
    length, n_new, keep_len = (torch.zeros(n_seq, **i32) for _ in range(3))
    parent, keep = torch.zeros(b.n_tokens, **i32), torch.zeros(b.n_tokens, **i32)
    qkv = torch.zeros(b.n_tokens, (hq + 2 * hkv) * dim, dtype=t, device="cuda")

    def step():
        plan = P.paged_plan(d, length, n_new, pool, held, table)
        tree = P.tree_mask(parent, plan.q_start, plan.kv_len, words)
        q = P.paged_append_rope(d, qkv, rope, table, plan.q_start, plan.kv_len, k, v, position=tree.position)
        o, lse = P.fa_tree(d, q, k, v, tree.mask, table, plan.q_start, plan.kv_len, ws=ws)
        attended = k.clone(), v.clone(), table.clone()
        P.paged_keep(d, k, v, keep, keep_len, table, plan.q_start, plan.kv_len, length=length)
        return q, o, lse, attended

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, o, lse, attended = step()
    rng = np.random.RandomState(hq)
    accepted = [[torch.zeros(0, hkv, dim, dtype=torch.float64, device="cuda")] * 2 for _ in range(n_seq)]   # rows of k, v
    missed = [[], []]
    for _ in range(steps):
        sizes = [int(n) for n in rng.randint(1, draft + 1, n_seq)]
        parents = [random_tree(rng, n, "any") for n in sizes]
        paths = []
        for p in parents:   # the way to a random token of the tree
            at, path = int(rng.randint(0, len(p))), []
            while at >= 0:
                path.append(at)
                at = int(p[at])
            paths.append(path[::-1])
        start, total = np.concatenate([[0], np.cumsum(sizes)]), sum(sizes)
        n_new.copy_(torch.tensor(sizes, **i32))
        parent[:total] = torch.tensor(np.concatenate(parents).tolist(), **i32)
        for s, path in enumerate(paths):
            keep[start[s]:start[s] + len(path)] = torch.tensor(path, **i32)
        keep_len.copy_(torch.tensor([len(p) for p in paths], **i32))
        qkv.copy_(torch.randn(qkv.shape, generator=b.gen, device="cuda").to(t))
        before = [len(r[0]) for r in accepted]
        graph.replay()
        P.check(P.device_error())
        # the cache as the attention saw it, with lengths and masks that this test keeps itself
        b.q_lens, b.kv_lens = sizes, [a + n for a, n in zip(before, sizes)]
        b.q_start_host = start.astype(np.int32)
        b.k, b.v, seen_table = attended
        b.table_host = seen_table.cpu().numpy()
        flat, depth = mask_of(parents, words)
        positions = np.zeros(b.n_tokens, np.int64)
        positions[:total] = np.repeat(before, sizes) + depth
        (want, size), (wk, ksize), wv = append64(b, qkv, kw, True, positions, None, None, 0.0)
        near(torch, t, q[:total], want[:total], size[:total])
        for s in range(n_seq):
            at = slice(int(start[s]), int(start[s + 1]))
            rows = b.rows(b.k, s), b.rows(b.v, s)
            assert all(torch.equal(x[:before[s]], y) for x, y in zip(rows, accepted[s])), "accepted rows"
            near(torch, t, rows[0][before[s]:], wk[at], ksize[at])
            assert torch.equal(rows[1][before[s]:], wv[at])
            taken = torch.tensor([before[s] + i for i in paths[s]], device="cuda")
            accepted[s] = [torch.cat([x[:before[s]], x[taken]]) for x in rows]
        bits = np.zeros((b.n_tokens, 32 * words), bool)
        bits[:total] = np.unpackbits(flat.view(np.uint8), axis=1, bitorder="little")
        bits = torch.from_numpy(bits).cuda()
        want = tree64(b, q, bits)
        check(torch, b, o, lse, want)
        # what the bound must not let through: no outputs at all, all of the tree seen
        missed[0].append(outside(torch, torch.zeros_like(o), want))
        missed[1].append(outside(torch, tree64(b, q, torch.ones_like(bits))[0].nan_to_num(), want))
        assert length.tolist() == [len(r[0]) for r in accepted]
    for s in range(n_seq):   # the rows that the last step kept
        b.kv_lens = [len(r[0]) for r in accepted]
        b.table_host = table.cpu().numpy()
        assert torch.equal(b.rows(k, s), accepted[s][0]) and torch.equal(b.rows(v, s), accepted[s][1])
    assert min(missed[0]) > 0.9, "the bound would take zeros"
    assert max(missed[1]) > 0.3, "the bound would take any mask"
