"""How many digits p100_fa_tree keeps of the probabilities, with fp32 outputs against 64 bits.

The bound of o is test_paged_digits_gpu's: (rel + 2 e + 2^-18) sum p |v| + tail sum |v| + 2^-24.  Up to 16 rows a kv head a
probability goes in two 16-bit parts, each rounded to nearest: rel = u^2 (2^-16 in bfloat16, 2^-22 in float16); larger
trees round it once, rel = u.  In float16 the largest probability is at least 2^7 and nothing below 2^-25 is held, so
tail = 2^-32; bfloat16 has FP32's range."""
import math

import numpy as np
import pytest

import p100_b200 as P
from test_draft_gpu import attend_tree, masks, tree64
from test_paged_gpu import Batch, check

pytestmark = pytest.mark.gpu


def worst(torch, b, q, bits, o, rel):
    """The largest error of o in units of its bound."""
    group, scale, most = b.hq // b.hkv, 1.0 / math.sqrt(b.dim), 0.0
    tail = 2.0 ** -32 if b.t == torch.float16 else 0.0
    for s, (n, t) in enumerate(zip(b.q_lens, b.kv_lens)):
        lo = int(b.q_start_host[s])
        seen = torch.ones(n, t, dtype=torch.bool, device="cuda")
        seen[:, t - n:] = bits[lo:lo + n, :n]
        k, v = b.rows(b.k, s), b.rows(b.v, s)
        for h in range(b.hq):
            qh, kh, vh = q[lo:lo + n, h].double(), k[:, h // group], v[:, h // group]
            e = (b.dim * 2.0 ** -24 * scale * (qh.abs() @ kh.abs().T) + 2.0 ** -20).masked_fill(~seen, 0.0)
            p = torch.softmax((qh @ kh.T * scale).masked_fill(~seen, -math.inf), 1)
            tol = (rel + 2 * e.amax(1, keepdim=True) + 2.0 ** -18) * (p @ vh.abs()) + tail * vh.abs().sum(0) + 2.0 ** -24
            most = max(most, float(((o[lo:lo + n, h].double() - p @ vh).abs() / tol).max()))
    return most


def digits(torch, q_lens, kv_lens, hq, hkv, dim, dtype, page, softcap=0.0):
    """(error in units of the bound of two parts, of one) of a batch of trees."""
    b = Batch(torch, q_lens, kv_lens, hq, hkv, dim, dtype, page, seed=70)
    b.fill()
    q = b.queries(3.0)
    mask, bits = masks(b, np.random.RandomState(0), "any", 1 + max(q_lens) // 32)
    # (a cap far above every score moves them by less than the bound's 2^-20, but takes the capped kernels)
    o, _ = P.fa_tree(b.desc(o_fp32=True, softcap=softcap), q, b.k, b.v, mask, b.table, b.q_start, b.kv_len)
    P.check(P.device_error())
    u = torch.finfo(b.t).eps / 2
    return worst(torch, b, q, bits, o, u * u), worst(torch, b, q, bits, o, u)


SMALL = [   # new tokens, query heads, kv heads: 1 to 16 rows of a kv head
    (1, 8, 1), (2, 8, 2), (8, 2, 2), (3, 3, 1), (2, 16, 2), (4, 8, 2), (16, 2, 2), (5, 3, 1), (13, 1, 1),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (128, 24)])
@pytest.mark.parametrize("n,hq,hkv", SMALL)
def test_digits_of_small_trees(cuda, n, hq, hkv, dim, page, dtype):
    """At most 16 rows of a kv head, on one CTA and cut over many: two parts."""
    for q_lens, kv_lens in (([n, 1, max(1, n - 1)], [n, 1 + 128, 700]), ([n], [3000])):
        two, _ = digits(cuda, q_lens, kv_lens, hq, hkv, dim, dtype, page)
        assert two <= 1.0, f"off by {two:.3g} of the bound"


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_digits_of_small_trees_under_a_cap(cuda, dtype):
    for n, hq, hkv in ((2, 16, 2), (3, 4, 1), (2, 4, 1)):
        two, _ = digits(cuda, [n, n], [700, 20], hq, hkv, 128, dtype, 16, softcap=1e6)
        assert two <= 1.0, f"off by {two:.3g} of the bound"


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,hq,hkv", [(2, 32, 4), (1, 12, 1), (16, 5, 5)])
def test_digits_of_many_small_trees(cuda, n, hq, hkv, dtype):
    """9 to 16 rows of a kv head in more row tiles than there are SMs."""
    sms = cuda.cuda.get_device_properties(0).multi_processor_count
    n_seq = -(-sms // hkv) + 1
    q_lens = [n] + [1 + i % n for i in range(n_seq - 1)]
    kv_lens = [m + i * 7 % 300 for i, m in enumerate(q_lens)]
    two, _ = digits(cuda, q_lens, kv_lens, hq, hkv, 128, dtype, 16)
    assert two <= 1.0, f"off by {two:.3g} of the bound"
    b = Batch(cuda, q_lens, kv_lens, hq, hkv, 128, dtype, 24, "token", seed=71, pad_rows=2, lead_rows=1)
    b.fill()
    q = b.queries()
    for kind, kw in (("bits", {}), ("empty", {}), ("any", dict(softcap=20.0, scale=-0.2))):
        mask, bits = masks(b, np.random.RandomState(1), kind, 1)
        check(cuda, b, *attend_tree(b, q, mask, **kw), tree64(b, q, bits, **kw))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,hq,hkv", [(17, 1, 1), (9, 4, 2), (40, 8, 1)])
def test_digits_of_larger_trees(cuda, n, hq, hkv, dim, dtype):
    """One rounding of each probability."""
    for q_lens, kv_lens in (([n, 1], [n, 700]), ([n], [3000])):
        _, one = digits(cuda, q_lens, kv_lens, hq, hkv, dim, dtype, 16)
        assert one <= 1.0, f"off by {one:.3g} of the bound"
