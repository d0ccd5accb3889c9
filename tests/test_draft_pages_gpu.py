"""Appends of tokens whose page lies outside the cache: what stays out of the pages, what is written all the same."""
import numpy as np
import pytest

import p100_b200 as P
from test_paged_gpu import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("computed", [True, False])
@pytest.mark.parametrize("bad", [-1, "n_pages", 2 ** 31 - 1, -2 ** 31])
@pytest.mark.parametrize("hq,hkv,dim,src,norm,half", [(2, 1, 64, "float32", False, False), (32, 8, 128, "bfloat16", True, True),
                                                      (5, 5, 128, "float16", True, False)])
def test_appends_to_pages_out_of_range(cuda, hq, hkv, dim, src, norm, half, bad, computed):
    """The tokens' keys and values reach no page and the flag is raised; their queries, and every other token's rows, are
    those of the call with a good table."""
    torch = cuda
    b = Batch(torch, [9, 3], [13, 7], hq, hkv, dim, "f16", 4, seed=5, lead_rows=1, pad_rows=1)
    qkv = torch.randn(b.n_tokens, (hq + 2 * hkv) * dim, generator=b.gen, device="cuda").to(getattr(torch, src))
    w = torch.rand(dim, generator=b.gen, device="cuda") + 0.5 if norm else None
    cs = torch.from_numpy(P.rope_table(16, dim, 10000.0)).cuda()

    def append(table, k, v):
        q = torch.full((b.n_tokens, hq, dim), 7.0, dtype=b.t, device="cuda")
        where = (table, b.q_start, b.kv_len, k, v)
        if computed:
            P.paged_append_rope(b.desc(), qkv, P.Rope(dim, 10000.0, half=half), *where, q_norm=w, k_norm=w, q=q)
        else:
            P.paged_append(b.desc(), qkv, *where, rope_cs=cs, rope_half=half, q_norm=w, k_norm=w, q=q)
        return q

    k, v = b.k.clone(), b.v.clone()
    want = append(b.table, k, v)
    P.check(P.device_error())
    table = b.table.clone()
    table[0, 2] = b.n_pages if bad == "n_pages" else bad   # tokens 8 to 11 of the first sequence: new ones 4 to 7
    got = append(table, b.k, b.v)
    with pytest.raises(P.InvalidArgument):
        P.check(P.device_error())
    assert torch.equal(got, want)
    page = int(b.table_host[0, 2])
    k[page], v[page] = np.nan, np.nan   # (as Batch leaves it)
    for x, y in ((b.k, k), (b.v, v)):
        assert torch.equal(x.view(torch.int16)[~torch.isnan(y)], y.view(torch.int16)[~torch.isnan(y)])
        assert torch.equal(torch.isnan(x), torch.isnan(y))
