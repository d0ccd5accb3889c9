"""Refusals of the paged-cache and scoring entry points: every argument check comes before any device call, so it
answers the same with and without a GPU; with valid arguments and no sm_100 device they return UNSUPPORTED."""
import ctypes as C
import math

import pytest

import p100_b200 as P
from test_capi import no_gpu

Z = C.c_void_p(256)


def desc(**kw):
    base = dict(n_seq=2, n_tokens=10, n_head_q=8, n_head_kv=2, page_size=16, n_pages=8, max_pages=4)
    return P.PagedDesc(**{**base, **kw})


def append(lib, d, qkv=Z, kind=P.F32, stride=0, norm=None, eps=1e-5, rope=None, max_pos=0):
    return lib.p100_paged_append(C.byref(d), qkv, kind, stride, norm, norm, eps, rope, max_pos, 0, Z, Z, Z, Z, Z, Z,
                                 None)


def attend(lib, d):
    return lib.p100_fa_paged(C.byref(d), Z, Z, Z, Z, Z, Z, Z, None, Z, 1 << 40, None)


@pytest.mark.parametrize("kw,why", [
    (dict(n_seq=-1), "counts must not be negative"),
    (dict(n_tokens=-1), "counts must not be negative"),
    (dict(max_q=-1), "counts must not be negative"),
    (dict(n_seq=P.PAGED_MAX_SEQ + 1), "n_seq exceeds P100_PAGED_MAX_SEQ"),
    (dict(n_head_q=0), "all dimensions must be positive"),
    (dict(page_size=0), "all dimensions must be positive"),
    (dict(n_head_q=7), "n_head_q must be divisible by n_head_kv"),
    (dict(head_dim=96), "head_dim must be 64 or 128"),
    (dict(dtype=P.F32), "dtype must be P100_F16 or P100_BF16"),
    (dict(scale=math.inf), "scale must be finite"),
    (dict(softcap=-1.0), "softcap must be finite and non-negative"),
    (dict(softcap=math.nan), "softcap must be finite and non-negative"),
    (dict(n_tokens=1 << 30), "n_tokens * n_head_q exceeds 2^31 - 1"),
    (dict(max_pages=1 << 30), "max_pages * page_size exceeds 2^31 - 1"),
    (dict(token_stride=64), "page strides must be at least head_dim"),
    (dict(head_stride=-128), "page strides must be at least head_dim"),
    (dict(page_stride=4100), "strides must be multiples of 8 elements"),
    (dict(q_stride=1000), "q and o strides must be at least n_head_q * head_dim"),
    (dict(o_stride=1028), "strides must be multiples of 8 elements"),
])
def test_descriptor_refusals(lib, kw, why):
    d = desc(**kw)
    for call in (append, attend):
        assert call(lib, d) == P.ERR_INVALID
        assert P.last_error() == why
    assert lib.p100_fa_paged_workspace_size(C.byref(d)) == 0
    assert P.last_error() == why


def test_append_refusals(lib):
    d = desc()
    for kw, why in ((dict(kind=7), "unknown qkv type 7"), (dict(stride=100), "qkv_stride must be at least a fused row"),
                    (dict(stride=1537), "qkv rows must be 16-byte aligned"),
                    (dict(norm=Z, eps=-1.0), "eps must be finite and non-negative"),
                    (dict(rope=Z, max_pos=0), "max_pos must be positive")):
        assert append(lib, d, **kw) == P.ERR_INVALID
        assert P.last_error() == why
    assert lib.p100_paged_append(None, Z, 0, 0, None, None, 0.0, None, 0, 0, Z, Z, Z, Z, Z, Z, None) == P.ERR_INVALID
    assert lib.p100_fa_paged(None, Z, Z, Z, Z, Z, Z, Z, None, Z, 1 << 40, None) == P.ERR_INVALID


def score(lib, dtype=P.F32, n=100, rows=2, stride=0, token=Z, k=3, lp=Z, rank=Z, index=Z, top=Z):
    return lib.p100_logprobs(Z, dtype, n, rows, stride, token, k, lp, Z, rank, index, top, None, 0, None)


def test_logprobs_refusals(lib):
    for kw, why in ((dict(dtype=5), "unknown logit type"), (dict(n=0), "rows must not be negative and n must be positive"),
                    (dict(rows=-1), "rows must not be negative and n must be positive"),
                    (dict(k=33), "top_k must be between 0 and 32"), (dict(k=-1), "top_k must be between 0 and 32"),
                    (dict(n=(1 << 24) + 1), "n exceeds 2^24"),
                    (dict(stride=99), "row_stride must be at least n"),
                    (dict(token=None), "logprob and rank need tokens"),
                    (dict(index=None), "top_k needs top_index and top_logprob")):
        assert score(lib, **kw) == P.ERR_INVALID
        assert P.last_error() == why
    assert lib.p100_logprobs_workspace_size(1, 0, P.F32, 0) == 0


@pytest.mark.skipif(not no_gpu(), reason="checks the behaviour without a GPU")
def test_unsupported_without_a_device(lib):
    assert append(lib, desc()) == P.ERR_UNSUPPORTED
    assert attend(lib, desc()) == P.ERR_UNSUPPORTED
    assert score(lib) == P.ERR_UNSUPPORTED
    assert lib.p100_fa_paged_workspace_init(Z, 256, None) == P.ERR_UNSUPPORTED
    assert lib.p100_logprobs_workspace_init(Z, 256, None) == P.ERR_UNSUPPORTED


@pytest.mark.gpu
def test_refusals_on_the_device(cuda, lib):
    """Null and misaligned buffers, small workspaces, tensors that are not where the call runs."""
    torch = cuda
    d = desc()
    size = lib.p100_fa_paged_workspace_size(C.byref(d))
    assert size > 0
    odd = C.c_void_p(264)
    assert lib.p100_fa_paged(C.byref(d), Z, Z, Z, None, Z, Z, Z, None, Z, size, None) == P.ERR_INVALID
    assert lib.p100_fa_paged(C.byref(d), odd, Z, Z, Z, Z, Z, Z, None, Z, size, None) == P.ERR_INVALID
    assert lib.p100_fa_paged(C.byref(d), Z, Z, Z, Z, Z, Z, Z, None, Z, size - 1, None) == P.ERR_INVALID
    assert lib.p100_fa_paged(C.byref(d), Z, Z, Z, Z, Z, Z, Z, None, None, size, None) == P.ERR_INVALID
    assert lib.p100_fa_paged(C.byref(d), Z, Z, Z, Z, Z, Z, Z, None, odd, size, None) == P.ERR_INVALID
    assert lib.p100_fa_paged(C.byref(d), Z, Z, Z, Z, Z, Z, Z, None, Z, size, None) == P.ERR_INVALID
    assert P.last_error() == "o must not be q"
    far = desc(n_tokens=1 << 27, max_q=1 << 27, n_head_q=8, page_size=9, max_pages=(1 << 31) // 9 - 1)
    assert lib.p100_fa_paged(C.byref(far), Z, Z, Z, Z, Z, Z, C.c_void_p(512), None, Z, size, None) == P.ERR_INVALID
    assert P.last_error() == "max_q x max_pages x page_size is too long for one call"
    assert append(lib, d, qkv=odd) == P.ERR_INVALID
    assert lib.p100_logprobs(C.c_void_p(258), P.F32, 100, 1, 0, None, 0, None, Z, None, None, None, None, 0,
                             None) == P.ERR_INVALID
    assert lib.p100_logprobs(Z, P.F32, 100000, 1, 0, None, 0, None, Z, None, None, None, None, 0, None) == P.ERR_INVALID
    # nothing to do is no error
    for kw in (dict(n_tokens=0), dict(n_seq=0)):
        assert attend(lib, desc(**kw)) == P.OK and append(lib, desc(**kw)) == P.OK
    assert score(lib, rows=0) == P.OK

    x = torch.zeros(10, 8, 128, dtype=torch.float16, device="cuda")
    pages = torch.zeros(8, 2, 16, 128, dtype=torch.float16, device="cuda")
    table = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 4, 10], dtype=torch.int32, device="cuda")
    lens = torch.tensor([4, 6], dtype=torch.int32, device="cuda")
    P.fa_paged(d, x, pages, pages, table, starts, lens)
    for bad in ((x.cpu(), pages, pages, table, starts, lens), (x.bfloat16(), pages, pages, table, starts, lens),
                (x[:9], pages, pages, table, starts, lens), (x, pages[:7].clone(), pages, table, starts, lens),
                (x, pages, pages, table.long(), starts, lens), (x, pages, pages, table[:1], starts, lens),
                (x, pages, pages, table, starts[:2], lens), (x, pages, pages, table, starts, lens.cpu()),
                (x.transpose(1, 2).contiguous().transpose(1, 2), pages, pages, table, starts, lens)):
        with pytest.raises(P.InvalidArgument):
            P.fa_paged(d, *bad)
    with pytest.raises(P.InvalidArgument):   # rows of the table that are longer than the descriptor's
        P.fa_paged(d, x, pages, pages, torch.zeros(2, 6, dtype=torch.int32, device="cuda"), starts, lens)
    with pytest.raises(P.InvalidArgument):
        P.fa_paged(d, x, pages, pages, table, starts, lens, o=x)
    with pytest.raises(P.InvalidArgument):   # a table of angles for another head size
        P.paged_append(d, torch.zeros(10, 1536, device="cuda"), table, starts, lens, pages, pages,
                       rope_cs=torch.zeros(64, 32, 2, device="cuda"))
    with pytest.raises(P.InvalidArgument):
        P.paged_append(d, torch.zeros(10, 1535, device="cuda"), table, starts, lens, pages, pages)
    with pytest.raises(P.InvalidArgument):
        P.paged_append(d, torch.zeros(10, 1536, device="cuda", dtype=torch.float64), table, starts, lens, pages, pages)
    for bad in (torch.zeros(4, 10), torch.zeros(10, device="cuda"), torch.zeros(10, 4, device="cuda").T,
                torch.zeros(4, 10, device="cuda", dtype=torch.int32)):
        with pytest.raises(P.InvalidArgument):
            P.logprobs(bad)
    with pytest.raises(P.InvalidArgument):
        P.logprobs(torch.zeros(4, 10, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(P.InvalidArgument):
        P.logprobs(torch.zeros(4, 10, device="cuda"), top_k=33)
    P.check(P.device_error())


@pytest.mark.gpu
def test_rows_that_overlap_are_refused(cuda):
    """Expanded rows have stride 0, which the C calls take for the contiguous default: refused before them."""
    torch = cuda
    d = desc()
    pages = torch.zeros(8, 2, 16, 128, dtype=torch.float16, device="cuda")
    table = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 4, 10], dtype=torch.int32, device="cuda")
    lens = torch.tensor([4, 6], dtype=torch.int32, device="cuda")
    with pytest.raises(P.InvalidArgument):
        P.logprobs(torch.zeros(1, 50, device="cuda").expand(4, 50))
    with pytest.raises(P.InvalidArgument):
        P.logprobs(torch.zeros(100, device="cuda").as_strided((4, 50), (8, 1)))
    with pytest.raises(P.InvalidArgument):
        P.paged_append(d, torch.zeros(1, 1536, device="cuda").expand(10, 1536), table, starts, lens, pages, pages)
    with pytest.raises(P.InvalidArgument):
        P.fa_paged(d, torch.zeros(1, 8, 128, dtype=torch.float16, device="cuda").expand(10, 8, 128), pages, pages,
                   table, starts, lens)
    with pytest.raises(P.InvalidArgument):
        P.fa_paged(d, torch.zeros((), dtype=torch.float16, device="cuda"), pages, pages, table, starts, lens)
    P.logprobs(torch.zeros(1, 50, device="cuda").expand(1, 50))
    P.check(P.device_error())
