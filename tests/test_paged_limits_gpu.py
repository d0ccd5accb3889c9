"""p100_fa_paged at the ends of what its descriptor takes, with the bounds of test_paged_gpu.py."""
import math

import pytest

from test_paged_gpu import Batch, attend, attend64, check

import p100_b200 as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("softcap,scale", [(1e-22, 1e-22), (3e-30, -1e-30), (1e-16, 2e-16), (1e-14, 1e-14)])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [300, 70]), ([90, 1], [300, 70])])
def test_tiny_caps_with_tiny_scales(cuda, q_lens, kv_lens, softcap, scale):
    """Every score is next to zero, so a row's visible keys weigh the same; hidden ones must not weigh anything, be the
    scores below half the cap (the polynomial's range) or beyond."""
    b = Batch(cuda, q_lens, kv_lens, 6, 2, 64, "bf16", 16, seed=60)
    b.fill()
    for size in (1.5, 0.01):
        q = b.queries(size)
        o, lse = attend(b, q, softcap=softcap, scale=scale, o_fp32=True)
        check(cuda, b, o, lse, attend64(b, q, scale, softcap))


@pytest.mark.parametrize("page,pages", [(8176, 262657), (114808, 18705)])   # 2^31 - 16 and 2^31 - 8 places
@pytest.mark.parametrize("n", [1, 5])
def test_as_many_keys_as_a_length_holds(cuda, n, page, pages):
    """A sequence of almost 2^31 tokens whose table names one page over and over.  Its keys are zero, so they weigh the same
    (V = 1); the newest token's own key (V = 3) decides its row and is hidden from the rows before it; what the page
    holds behind the last token would decide every row if it took part.

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
    o, lse = P.fa_paged(d, q, k, v, table, torch.tensor([0, n], dtype=torch.int32, device="cuda"),
                        torch.tensor([kv], dtype=torch.int32, device="cuda"))
    P.check(P.device_error())
    x = 5.0 * dim / math.sqrt(dim)   # the newest key's score; the others' weight is below 2^31 e^-40 < 2^-26 of its own
    assert bool(((o[:-1] - 1.0).abs() <= 2.0 ** -14).all())
    assert bool(((o[-1] - 3.0).abs() <= 3 * 2.0 ** -14).all())
    assert bool(((lse[:-1] - math.log(kv)).abs() <= 2.0 ** -14 + 2.0 ** -22 * math.log(kv)).all())
    assert bool(((lse[-1] - x).abs() <= 2.0 ** -14 + 2.0 ** -22 * x).all())
