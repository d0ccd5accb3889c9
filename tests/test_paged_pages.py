"""The Python binding's check of page tensors: sizes that name the axes come with the descriptor's strides."""
import pytest
import torch

import p100_b200 as P

HOST = -1   # the device that a tensor in host memory reports


def desc(**kw):
    return P.PagedDesc(n_seq=1, n_tokens=1, n_head_q=6, n_head_kv=kw.pop("heads", 3), page_size=16, n_pages=5,
                       max_pages=5, head_dim=64, **kw)


def pages(*shape):
    return torch.zeros(shape, dtype=torch.float16)


BY_TOKEN = dict(head_stride=64, token_stride=3 * 64)


def test_layouts_that_fit():
    heads, tokens = pages(5, 3, 16, 64), pages(5, 16, 3, 64)
    for t, kw in ((heads, {}), (tokens, BY_TOKEN), (tokens.transpose(1, 2), BY_TOKEN), (heads.transpose(1, 2), {}),
                  (pages(5, 2, 3, 16, 64)[:, 1], dict(page_stride=2 * 3 * 16 * 64)),
                  (pages(5, 2, 16, 3, 64)[:, 0], dict(page_stride=2 * 3 * 16 * 64, **BY_TOKEN)),
                  (pages(9, 3, 16, 64), {}), (pages(5 * 3 * 16 * 64), {}), (pages(5, 3 * 16 * 64), {}),
                  (pages(5, 2, 3, 16, 64), dict(page_stride=2 * 3 * 16 * 64)), (pages(5, 16, 64), dict(heads=1)),
                  (pages(5, 1, 16, 64), dict(heads=1)), (pages(5, 16, 1, 64), dict(heads=1))):
        P._pages_of(t, t, HOST, desc(**kw))


def test_layouts_that_the_kernel_would_misread():
    heads, tokens = pages(5, 3, 16, 64), pages(5, 16, 3, 64)
    good = {(): heads, tuple(BY_TOKEN): tokens}
    for t, kw in ((tokens, {}), (heads, BY_TOKEN), (tokens.transpose(1, 2), {}), (heads.transpose(1, 2), BY_TOKEN),
                  (pages(5, 2, 3, 16, 64)[:, 1], {}), (heads, dict(page_stride=2 * 3 * 16 * 64)),
                  (pages(5, 3, 64, 16).transpose(2, 3), {}), (pages(1, 3, 16, 64).expand(5, 3, 16, 64), {})):
        for args in ((t, good[tuple(BY_TOKEN) if "token_stride" in kw else ()]), (good[()], t)):
            with pytest.raises(P.InvalidArgument, match="has strides"):
                P._pages_of(*args, HOST, desc(**kw))
    t = pages(5, 2, 16, 64)[:, 0]
    with pytest.raises(P.InvalidArgument, match="has strides"):
        P._pages_of(t, t, HOST, desc(heads=1))


@pytest.mark.gpu
def test_calls_refuse_them(cuda):
    d = desc()
    ints = lambda *v: cuda.tensor(v, dtype=cuda.int32, device="cuda")
    good, bad = pages(5, 3, 16, 64).cuda(), pages(5, 16, 3, 64).cuda()
    lengths = (ints(0, 1, 2, 3, 4).view(1, 5), ints(0, 1), ints(1))
    for k, v in ((good, bad), (bad, good)):
        with pytest.raises(P.InvalidArgument, match="has strides"):
            P.paged_append(d, cuda.zeros(1, 12 * 64, device="cuda"), *lengths, k, v)
        with pytest.raises(P.InvalidArgument, match="has strides"):
            P.fa_paged(d, pages(1, 6, 64).cuda(), k, v, *lengths)
