"""A step over the paged cache whose plan finds too few pages, and the lengths that p100_paged_keep leaves in every case."""
import numpy as np
import pytest

import p100_b200 as P
from test_draft_gpu import random_tree

pytestmark = pytest.mark.gpu


def small_step(torch, n_pages, dtype=P.F16):
    """(descriptor, state, step()) of three requests of up to 9 new tokens over pages of 4; step() goes from the plan to the
    kept rows and returns (plan, q, o, lse)."""
    n_seq, draft, hq, hkv, dim = 3, 9, 4, 2, 64
    i32 = dict(dtype=torch.int32, device="cuda")
    d = P.PagedDesc(n_seq=n_seq, n_tokens=n_seq * draft, max_q=draft, n_head_q=hq, n_head_kv=hkv, page_size=4,
                    n_pages=n_pages, max_pages=8, head_dim=dim, dtype=dtype)
    pool, held, table = P.paged_pool(d)
    s = dict(pool=pool, held=held, table=table, length=torch.zeros(n_seq, **i32), n_new=torch.zeros(n_seq, **i32),
             parent=torch.arange(n_seq * draft, **i32) * 0 - 1, keep=torch.zeros(n_seq * draft, **i32),
             keep_len=torch.zeros(n_seq, **i32))
    s["k"] = torch.randn((n_pages, hkv, 4, dim), device="cuda").half()
    s["v"] = torch.randn((n_pages, hkv, 4, dim), device="cuda").half()
    s["qkv"] = torch.randn(d.n_tokens, (hq + 2 * hkv) * dim, device="cuda")
    s["q"] = torch.zeros(d.n_tokens, hq, dim, dtype=torch.float16, device="cuda")
    s["o"], s["lse"] = torch.zeros_like(s["q"]), torch.zeros(d.n_tokens, hq, device="cuda")
    rope, ws = P.Rope(dim, 10000.0), P.fa_paged_workspace(d)

    def step(length=None):
        plan = P.paged_plan(d, s["length"], s["n_new"], pool, held, table)
        tree = P.tree_mask(s["parent"], plan.q_start, plan.kv_len, 1)
        where = (table, plan.q_start, plan.kv_len)
        P.paged_append_rope(d, s["qkv"], rope, *where, s["k"], s["v"], position=tree.position, q=s["q"])
        P.fa_tree(d, s["q"], s["k"], s["v"], tree.mask, *where, o=s["o"], lse=s["lse"], ws=ws)
        return P.paged_keep(d, s["k"], s["v"], s["keep"], s["keep_len"], *where, length=length)

    return d, s, step


@pytest.mark.parametrize("captured", [False, True])
def test_a_step_without_enough_pages_does_nothing(cuda, captured):
    """The caller asks to keep drafts that the plan had no pages for: nothing is written, no flag is raised, the lengths stay,
    and the next step, which has pages, goes on from them."""
    torch = cuda
    d, s, step = small_step(torch, 6)
    P.check(P.device_error())
    run = step
    if captured:
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step(s["length"])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(s["length"])

        def run(length):   # noqa: F811
            graph.replay()
            return length

    def numbers(name, values):
        s[name].copy_(torch.tensor(values, dtype=torch.int32))

    numbers("n_new", [9, 5, 2])   # 3 + 2 + 1 pages: all of the pool
    numbers("keep", [0, 1, 2, 0, 0, 0, 0, 0, 0, 0, 1, 0, 0, 0, 0, 1] + [0] * 11)
    numbers("keep_len", [3, 2, 2])
    run(s["length"])
    P.check(P.device_error())
    assert s["length"].tolist() == [3, 2, 2]
    numbers("n_new", [9, 9, 9])
    names = ("k", "v", "q", "o", "lse", "held", "table")
    before = {n: s[n].clone() for n in names}
    for asked in ([3, 2, 2], [0, 9, 1], [9, 9, 9]):
        numbers("keep_len", asked)
        got = run(s["length"])
        P.check(P.device_error())
        assert int(s["pool"][1]) == 3 and got.tolist() == s["length"].tolist() == [3, 2, 2]
        assert all(torch.equal(s[n], before[n]) for n in names)
    if not captured:   # a length that the call allocates
        assert step().tolist() == [3, 2, 2]
        P.check(P.device_error())
    numbers("n_new", [1, 1, 1])
    numbers("keep_len", [1, 1, 1])
    numbers("keep", [0] * 27)
    run(s["length"])
    P.check(P.device_error())
    assert int(s["pool"][1]) == 0 and s["length"].tolist() == [4, 3, 3]


@pytest.mark.parametrize("dim,hkv", [(64, 1), (128, 12)])   # one block a sequence, and several
def test_keep_gives_every_sequence_a_length(cuda, dim, hkv):
    """Counts out of range keep nothing; a sequence whose starts or length are out of range is left as it was.  Both raise
    the flag, and no sequence moves a row that it should not."""
    torch = cuda
    i32 = dict(dtype=torch.int32, device="cuda")
    d = P.PagedDesc(n_seq=3, n_tokens=12, n_head_q=hkv, n_head_kv=hkv, page_size=4, n_pages=15, max_pages=5, head_dim=dim)
    table = torch.arange(15, **i32).view(3, 5)
    keep = torch.tensor([1, 2, 3, 0] * 3, **i32)
    for start, kv, count, want, moves in (
            ([0, 4, 8, 12], [10, 11, 12], [2, 5, -1], [8, 7, 8], [0]),          # counts behind n and below 0
            ([0, 4, 4, 8], [10, 11, 12], [0, 7, 1], [6, 11, 9], [2]),           # no new tokens: the count is not looked at
            ([0, 4, 8, 13], [10, 11, 12], [1, 1, 1], [7, 8, 12], [0, 1]),       # tokens behind n_tokens
            ([0, 4, 3, 7], [10, 11, 12], [1, 1, 1], [7, 11, 9], [0]),           # starts that fall (then keep[3] = 0: it stays)
            ([-1, 4, 8, 12], [10, 11, 12], [1, 1, 1], [10, 8, 9], [1, 2]),      # a negative one
            ([0, 4, 8, 12], [3, 21, 12], [1, 1, 4], [3, 21, 12], [2]),          # fewer tokens than new ones; more than the table
            ([0, 4, 8, 12], [10, -5, 12], [1, 0, 0], [7, -5, 8], [0])):
        k = torch.randn(15, hkv, 4, dim, device="cuda").half()
        v = torch.randn(15, hkv, 4, dim, device="cuda").half()
        rows = [x.clone() for x in (k, v)]
        length = torch.full((3,), 77, **i32)
        where = (table, torch.tensor(start, **i32), torch.tensor(kv, **i32))
        P.paged_keep(d, k, v, keep, torch.tensor(count, **i32), *where, length=length)
        torch.cuda.synchronize()
        flagged = P.device_error() != 0
        assert length.tolist() == want, (start, kv, count)
        assert flagged == (start != [0, 4, 4, 8])
        for x, old in zip((k, v), rows):
            for s in range(3):
                new, was = (y[5 * s:5 * s + 5].permute(0, 2, 1, 3).reshape(20, hkv, dim) for y in (x, old))
                should = was.clone()
                if s in moves:
                    ctx = kv[s] - 4
                    for i in range(count[s]):
                        if i < 3:   # keep[3] = 0 is out of order
                            should[ctx + i] = was[ctx + i + 1]
                assert torch.equal(new, should), (start, kv, count, s)
