"""p100_logprobs on the GPU against 64 bits.

Tolerances.  FP32 sums of at most 200,000 positive terms, each thread's chain below 2^9 terms and joined in a tree:
relative error below 2^9 2^-24 + the exponentials' 2^-21, so ln s is off by less than 2^-14 in the worst case and the
differences x - m - ln s by that plus 2^-23 of their size.  The entropy's u / s carries the same relative error."""
import math

import numpy as np
import pytest

import p100_b200 as P

pytestmark = pytest.mark.gpu


def want(torch, x, tokens, k):
    """The definition in 64 bits: masked logits (-inf, NaN) have probability 0 and are no alternatives."""
    y = torch.where(torch.isnan(x.double()), torch.full_like(x, -math.inf, dtype=torch.float64), x.double())
    m = y.amax(1, keepdim=True)
    none = torch.isneginf(m)
    e = torch.where(none, torch.zeros_like(y), torch.exp(y - torch.where(none, torch.zeros_like(m), m)))
    s = e.sum(1, keepdim=True)
    # relative to m, which may be so large that m + ln s is m
    y, y0 = torch.where(none, y, y - torch.where(none, torch.zeros_like(m), m)), y
    lse = torch.where(none, torch.zeros_like(m), s.clamp(min=1e-300).log())
    p = torch.where(none, torch.zeros_like(e), e / s.clamp(min=1e-300))
    ent = -torch.where(p > 0, p * (y - lse), torch.zeros_like(y)).sum(1)
    tok = tokens.long().clamp(min=0)[:, None]
    xt = y.gather(1, tok)
    lp = (xt - lse)[:, 0]
    idx = torch.arange(x.shape[1], device=x.device)
    real = ~torch.isnan(x.double())
    x0 = y0.gather(1, tok)
    rank = (real & ((y0 > x0) | ((y0 == x0) & (idx < tok)))).sum(1).int()
    lp = torch.where(tokens < 0, torch.zeros_like(lp), lp)
    rank = torch.where(tokens < 0, torch.full_like(rank, -1), rank)
    v, at = torch.sort(y, dim=1, descending=True, stable=True)
    v, at = v[:, :k], at[:, :k].int()
    if v.shape[1] < k:
        pad = k - v.shape[1]
        v = torch.cat([v, torch.full((x.shape[0], pad), -math.inf, dtype=torch.float64, device=x.device)], 1)
        at = torch.cat([at, torch.full((x.shape[0], pad), -1, dtype=torch.int32, device=x.device)], 1)
    at = torch.where(torch.isneginf(v), torch.full_like(at, -1), at)
    return lp, ent, rank, at, v - lse


def close(torch, got, ref, what):
    got = got.double()
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf]), what
    d = (got - ref)[~inf].abs()
    tol = 2.0 ** -14 + 2.0 ** -22 * ref[~inf].abs()
    assert bool((d <= tol).all()), f"{what} off by {float(d.max()):.3g}"


def check(torch, x, tokens, k, **kw):
    r = P.logprobs(x, tokens, top_k=k, **kw)
    P.check(P.device_error())
    lp, ent, rank, at, top = want(torch, x, tokens, k)
    close(torch, r.logprob, lp, "logprob")
    close(torch, r.entropy, ent, "entropy")
    assert torch.equal(r.rank, rank)
    assert torch.equal(r.top_index, at)
    close(torch, r.top_logprob, top, "top_logprob")
    return r


def logits(torch, rows, n, dtype, seed, scale=3.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(rows, n, generator=g, device="cuda") * scale).to(getattr(torch, dtype))


def some_tokens(torch, rows, n, seed=0):
    return torch.from_numpy(np.random.RandomState(seed).randint(0, n, rows).astype(np.int32)).cuda()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 128256, 20), (3, 2, 5), (7, 31, 32), (2, 4097, 0), (5, 32003, 32),
                                      (230, 5001, 3), (500, 777, 8), (1, 200001, 32), (40, 12345, 1)])
def test_rows(cuda, rows, n, k, dtype):
    x = logits(cuda, rows, n, dtype, rows + n)
    check(cuda, x, some_tokens(cuda, rows, n), k)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_ties_go_to_the_lowest_index(cuda, dtype):
    """Rows of few distinct values: more equals than the candidates' buffer holds, at both ends of a row."""
    x = logits(cuda, 6, 30011, dtype, 1, 0.4).round()
    x[0] = 2.0
    x[1, :] = -1.0
    x[1, -1] = 5.0
    x[2, 10000:] = 9.0
    check(cuda, x, some_tokens(cuda, 6, 30011, 3), 32)


@pytest.mark.parametrize("n", [33, 130, 600, 1025, 9000, 70001])
@pytest.mark.parametrize("k", [1, 7, 32])
def test_equal_logits(cuda, n, k):
    """Equal rows, and rows with a finite value in their masked places: few to many candidates of one value."""
    x = cuda.zeros(3, n, device="cuda")
    x[1] = -1e4
    x[1, 5:9] = 1.0
    x[2, ::2] = 3.5
    r = check(cuda, x, some_tokens(cuda, 3, n, 6), k)
    assert r.top_index[0].tolist() == list(range(k))


def test_masked_rows(cuda):
    """-inf, NaN and the type's lowest value; a row with nothing, one with one logit, fewer than top_k."""
    for dtype in ("float32", "float16", "bfloat16"):
        x = logits(cuda, 8, 5003, dtype, 2)
        lowest = cuda.finfo(x.dtype).min
        x[0] = -math.inf
        x[1] = -math.inf
        x[1, 4000] = 1.5
        x[2, 1::2] = math.nan
        x[3] = lowest
        x[4, 7:] = lowest
        x[5, 5:] = -math.inf
        x[6] = math.nan
        tokens = some_tokens(cuda, 8, 5003, 4)
        tokens[1] = 4000
        tokens[2] = 2000
        tokens[3] = 17
        tokens[4] = 3
        tokens[5] = 1
        tokens[7] = -1
        check(cuda, x, tokens, 12)


def test_tokens_that_are_masked_or_missing(cuda):
    x = logits(cuda, 4, 1000, "float32", 3)
    x[0, 10] = -math.inf
    x[1, 20] = -math.inf
    x[1, 5] = -math.inf
    tokens = cuda.tensor([10, 20, -1, 999], dtype=cuda.int32, device="cuda")
    check(cuda, x, tokens, 2)
    r = P.logprobs(x, cuda.tensor([1000, -2, 0, 1], dtype=cuda.int32, device="cuda"))
    with pytest.raises(P.InvalidArgument):
        P.check(P.device_error())
    assert r.logprob[:2].tolist() == [0.0, 0.0] and r.rank[:2].tolist() == [-1, -1]
    r = P.logprobs(x, top_k=2)
    assert r.logprob is None and r.rank is None
    assert cuda.equal(r.top_index, want(cuda, x, tokens, 2)[3])


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_masked_logits_that_start_late(cuda, dtype):
    """A padded vocabulary, and single masked logits far into rows that begin without any."""
    x = logits(cuda, 6, 70001, dtype, 6)
    x[0, 69000:] = -math.inf
    x[1, 40000] = -math.inf
    x[2, 50001] = math.nan
    x[3, 30000:] = cuda.finfo(x.dtype).min
    x[4, 20000::7] = -math.inf
    x[5, 69999:] = math.nan
    tokens = some_tokens(cuda, 6, 20000, 7)
    check(cuda, x, tokens, 16)
    check(cuda, x[1:2], tokens[1:2], 16)


def test_rows_beyond_32_bits(cuda):
    """Rows 400 MB apart: the last starts 2.2 billion elements behind the first."""
    gap, rows, n = 200_000_003, 12, 5003
    store = cuda.empty((rows - 1) * gap + n, dtype=cuda.float16, device="cuda")
    x = store.as_strided((rows, n), (gap, 1))
    x.copy_(logits(cuda, rows, n, "float16", 8))
    check(cuda, x, some_tokens(cuda, rows, n, 8), 4)


def test_infinite_logit(cuda):
    x = logits(cuda, 2, 3000, "float32", 4)
    x[0, 77] = math.inf
    r = P.logprobs(x, some_tokens(cuda, 2, 3000), top_k=2)
    P.check(P.device_error())
    assert math.isnan(float(r.logprob[0])) and math.isnan(float(r.entropy[0]))
    assert int(r.top_index[0, 0]) == 77 and not math.isnan(float(r.logprob[1]))


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_strided_unaligned_rows(cuda, dtype, offset):
    """Rows that start off every vector boundary, inside wider ones."""
    wide = cuda.full((9, 2100), 100.0, dtype=getattr(cuda, dtype), device="cuda")
    x = wide[:, offset:offset + 2051]
    x.copy_(logits(cuda, 9, 2051, dtype, 5))
    check(cuda, x, some_tokens(cuda, 9, 2051), 7)
    check(cuda, x[:1], some_tokens(cuda, 1, 2051), 7)


def test_sharp_and_flat_rows(cuda):
    x = cuda.zeros(3, 50000, device="cuda")
    x[1] = cuda.linspace(-400.0, 400.0, 50000, device="cuda")
    x[2] = 3000.0
    x[2, 123] = 3020.0
    check(cuda, x, some_tokens(cuda, 3, 50000), 5)


@pytest.mark.parametrize("dtype,base,step,n", [("float32", 1e6 / 3, 0.25, 5003), ("float32", -7.7e6, 1.0, 301),
                                               ("float16", 50016.0, 32.0, 4097), ("bfloat16", 3.1e5, 2048.0, 700),
                                               ("bfloat16", -3.3e30, 2.0 ** 95, 129), ("float32", 1.7e37, 2.0 ** 101, 65)])
def test_large_logits(cuda, dtype, base, step, n):
    """A common offset changes nothing: the differences are exact, so the tolerance has no term in the offset's size."""
    g = cuda.Generator(device="cuda")
    g.manual_seed(n)
    y = cuda.randint(-6, 7, (5, n), generator=g, device="cuda").double() * step
    x = (y + base).to(getattr(cuda, dtype))
    check(cuda, x, some_tokens(cuda, 5, n, 9), 4)


def test_confident_rows(cuda):
    """One logit far above the rest: the small log probability of the top and the entropy keep their digits.  Terms of
    e^-d carry 2^-22 and d's rounding, 2^-24 d; s = 1 + sum is rounded to 2^-24, and so are ln s and the entropy."""
    for dtype, top in (("float32", 31.7), ("float16", 29.3), ("bfloat16", 33.25)):
        x = logits(cuda, 16, 3001, dtype, 5, 1.0)
        x[:, 77] = top
        x[8:, 5:70] = -math.inf
        tokens = cuda.full((16,), 77, dtype=cuda.int32, device="cuda")
        r = check(cuda, x, tokens, 1)
        lp, ent = want(cuda, x, tokens, 1)[:2]
        assert float((r.logprob.double() - lp).abs().max()) <= 2.0 ** -22
        assert float((r.entropy.double() - ent).abs().max()) <= 2.0 ** -22


def test_graph_stream_and_shared_workspace(cuda):
    """One workspace for calls of several shapes, the same bits on every run, a captured call on new logits."""
    torch = cuda
    ws = P.logprobs_workspace(200, 9000, 32)
    for rows, n, k in ((1, 9000, 32), (200, 9000, 5), (3, 9000, 0), (150, 4000, 8), (1, 9000, 20)):
        x = logits(torch, rows, n, "float32", rows)
        check(torch, x, some_tokens(torch, rows, n), k, ws=ws)
    x = logits(torch, 2, 9000, "float32", 9)
    tokens = some_tokens(torch, 2, 9000)
    a = P.logprobs(x, tokens, top_k=20, ws=ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    b = P.logprobs(x, tokens, top_k=20, stream=side)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c = P.logprobs(x, tokens, top_k=20, ws=ws)
    x.copy_(logits(torch, 2, 9000, "float32", 10))
    graph.replay()
    torch.cuda.synchronize()
    lp, ent, rank, at, top = want(torch, x, tokens, 20)
    assert torch.equal(c.top_index, at) and torch.equal(c.rank, rank)
    close(torch, c.logprob, lp, "logprob")
