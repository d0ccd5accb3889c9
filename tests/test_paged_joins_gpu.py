"""p100_fa_paged where many CTAs share a row tile: single tokens over long contexts on few kv heads, whose parts are
joined in groups, against the 64-bit restatement and the bounds of test_paged_gpu.py.  Every call has outputs filled
with NaN before it and leaves the workspace's tickets at zero."""
import math
import random

import pytest

from test_paged_gpu import Batch, attend64, check
from test_paged_joins import FOLLOWED

import p100_b200 as P

pytestmark = pytest.mark.gpu


def serve(torch, b, q, want, ws, **kw):
    """One call on workspace ws, checked; the outputs."""
    o = torch.full((b.n_tokens, b.hq, b.dim), math.nan, dtype=b.t, device="cuda")
    lse = torch.full((b.n_tokens, b.hq), math.nan, device="cuda")
    P.fa_paged(b.desc(**kw), q, b.k, b.v, b.table, b.q_start, b.kv_len, o=o, lse=lse, ws=ws)
    P.check(P.device_error())
    check(torch, b, o, lse, want)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert not bool(ws.view(torch.int32)[:sms * 4].any()), "tickets are not zero"
    return o, lse


def workspace(b):
    return P.fa_paged_workspace(b.desc())


def batch(torch, lens, kv_heads, group, dtype, dim, page, seed, q_lens=None):
    b = Batch(torch, q_lens or [1] * len(lens), lens, kv_heads * group, kv_heads, dim, dtype, page, seed=seed, spare=0)
    b.fill()
    return b, b.queries()


def short_call(torch, ws, kv_heads, group, dtype, dim):
    b, q = batch(torch, [700, 5, 2049], kv_heads, group, dtype, dim, 16, 99)
    serve(torch, b, q, attend64(b, q), ws)


@pytest.mark.parametrize("heads,lens", FOLLOWED)
def test_tile_behind_a_group_of_one_part(cuda, heads, lens):
    b, q = batch(cuda, lens, heads, 8, "f16", 128, 64, len(lens))
    want, ws = attend64(b, q), workspace(b)
    first = serve(cuda, b, q, want, ws)
    for _ in range(20):
        again = serve(cuda, b, q, want, ws)
        assert all(cuda.equal(x, y) for x, y in zip(first, again))
    short_call(cuda, ws, heads, 8, "f16", 128)


@pytest.mark.parametrize("seed", range(12))
def test_ragged_long_contexts(cuda, seed):
    """Batches that mix long and short sequences on 1, 2 and 4 kv heads; up to four new tokens of a sequence."""
    rng = random.Random(seed)
    heads, group, dtype, dim = (1, 2, 4)[seed % 3], rng.choice([1, 4, 8, 16]), rng.choice(["f16", "bf16"]), rng.choice([64, 128])
    lens = [rng.randint(20000, 60000)] + [int(2 ** rng.uniform(0, 16)) for _ in range(rng.randint(1, 5))]
    rng.shuffle(lens)
    q_lens = [min(t, rng.randint(1, max(1, min(4, 16 // group)))) for t in lens]
    b, q = batch(cuda, lens, heads, group, dtype, dim, rng.choice([16, 24, 64, 256]), seed, q_lens)
    want, ws = attend64(b, q), workspace(b)
    first = serve(cuda, b, q, want, ws)
    for _ in range(5):
        again = serve(cuda, b, q, want, ws)
        assert all(cuda.equal(x, y) for x, y in zip(first, again))
    short_call(cuda, ws, heads, group, dtype, dim)


@pytest.mark.parametrize("parts", [2, 47, 48, 49, 50, 56, 57, 58, 64, 65, 73, 100, 183, 211, 295])
def test_numbers_of_parts(cuda, parts):
    """One sequence on one kv head in shares of two units: as many parts as are joined at once, and several groups with
    a last one of one, some or as many parts as the others."""
    b, q = batch(cuda, [64 * (2 * parts - 1) - 3], 1, 4, "bf16", 64, 16, parts)
    ws = workspace(b)
    for causal in (True, False):
        serve(cuda, b, q, attend64(b, q, causal=causal), ws, causal=causal)


def test_parts_of_chunks(cuda):
    """The tcgen05 kernel's cut tiles: short chunks over long contexts, two and more parts, the second rows' group."""
    b, q = batch(cuda, [40000, 300, 9000], 2, 5, "f16", 64, 32, 7, [40, 60, 90])
    want, ws = attend64(b, q), workspace(b)
    first = serve(cuda, b, q, want, ws)
    again = serve(cuda, b, q, want, ws)
    assert all(cuda.equal(x, y) for x, y in zip(first, again))


def test_replayed_with_other_lengths_beside_another_call(cuda):
    """A captured call of several levels whose lengths change between replays, while another stream runs the same
    sequences with a workspace of its own."""
    torch = cuda
    heads, lens = FOLLOWED[0]
    b, q = batch(torch, lens, heads, 8, "f16", 128, 64, 3)
    ws, other = workspace(b), workspace(b)
    o = torch.empty((b.n_tokens, b.hq, b.dim), dtype=b.t, device="cuda")
    lse = torch.empty((b.n_tokens, b.hq), device="cuda")
    o2, lse2 = torch.empty_like(o), torch.empty_like(lse)
    args = (b.desc(), q, b.k, b.v, b.table, b.q_start, b.kv_len)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        P.fa_paged(*args, o=o, lse=lse, ws=ws)
    side = torch.cuda.Stream()
    for kv in (lens, [lens[0] - 64, 200], [9000, 1], lens):
        b.kv_lens = kv
        b.kv_len.copy_(torch.tensor(kv, dtype=torch.int32))
        want = attend64(b, q)
        for x in (o, lse, o2, lse2):
            x.fill_(math.nan)
        torch.cuda.synchronize()
        for _ in range(10):
            graph.replay()
            P.fa_paged(*args, o=o2, lse=lse2, ws=other, stream=side)
        torch.cuda.synchronize()
        P.check(P.device_error())
        check(torch, b, o, lse, want)
        assert torch.equal(o, o2) and torch.equal(lse, lse2)
