"""Plans whose rows or pages are as many as 32 bits count."""
import pytest

import p100_b200 as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_new", [5, 2 ** 31 - 3])   # the second one is refused: too few pages
def test_plan_of_as_many_rows_as_32_bits_count(cuda, n_new):
    """2^31 - 1 rows: those behind the new tokens get -1, and nothing is written elsewhere."""
    torch = cuda
    n, i32 = 2 ** 31 - 1, dict(dtype=torch.int32, device="cuda")
    d = P.PagedDesc(n_seq=1, n_tokens=n, n_head_q=1, n_head_kv=1, page_size=1 << 20, n_pages=4, max_pages=2047)
    pool, held, table = P.paged_pool(d)
    around = torch.full((n + 2 * 65536,), 7, **i32)
    out = P.PagedPlan(torch.zeros(2, **i32), torch.zeros(1, **i32), None, around[65536:65536 + n])
    if n_new > 2047 << 20:
        n_new = 2047 << 20
    P.paged_plan(d, torch.tensor([0], **i32), torch.tensor([n_new], **i32), pool, held, table, out=out)
    P.check(P.device_error())
    got = n_new if n_new == 5 else 0
    assert int(pool[1]) == (0 if got else 2043)
    assert out.q_start.tolist() == [0, got] and out.position[:got].tolist() == list(range(got))
    assert bool((out.position[got:1 << 20] == -1).all())
    assert int(out.position[got:].max()) == -1 and int(out.position[got:].min()) == -1
    assert bool((around[:65536] == 7).all()) and bool((around[65536 + n:] == 7).all())


def test_plan_of_as_many_pages_as_32_bits_count(cuda):
    """A request that takes 2^31 - 9 pages of one token at once and gives them back."""
    torch = cuda
    n, i32 = 2 ** 31 - 9, dict(dtype=torch.int32, device="cuda")
    d = P.PagedDesc(n_seq=1, n_tokens=5000, n_head_q=1, n_head_kv=1, page_size=1, n_pages=n, max_pages=n)
    pool, held, table = P.paged_pool(d)
    zero = torch.zeros(1, **i32)
    P.paged_plan(d, torch.tensor([n], **i32), zero, pool, held, table)
    P.check(P.device_error())
    assert pool[:2].tolist() == [0, 0] and held.tolist() == [n]
    for at in (0, 1, 12345, n // 2, n - 8193, n - 8192, n - 1):
        assert int(table[0, at]) == at
    P.paged_plan(d, zero, zero, pool, held, table)
    P.check(P.device_error())
    assert pool[:2].tolist() == [n, 0] and held.tolist() == [0]
    assert int(table.max()) == -1
    for at in (0, 1, 12345, n // 2, n - 8193, n - 8192, n - 1):
        assert int(pool[2 + at]) == n - 1 - at
