"""Refusals of the entry points for steps and drafted trees, with and without a GPU, and the rotary frequencies, which
are computed on the host."""
import ctypes as C
import math

import numpy as np
import pytest

import p100_b200 as P
from test_capi import no_gpu
from test_serve_capi import desc

Z = C.c_void_p(256)


def plan(lib, d):
    return lib.p100_paged_plan(C.byref(d), *[Z] * 9, None)


def append(lib, d, rope=None, kind=P.F32, stride=0, norm=None, eps=1e-5):
    rope = P.Rope(64, 10000.0) if rope is None else rope
    return lib.p100_paged_append_rope(C.byref(d), Z, kind, stride, norm, norm, eps, C.byref(rope), *[Z] * 7, None)


def tree(lib, d, words=1):
    return lib.p100_fa_tree(C.byref(d), Z, Z, Z, Z, words, Z, Z, Z, Z, None, Z, 1 << 40, None)


def keep(lib, d):
    return lib.p100_paged_keep(C.byref(d), *[Z] * 8, None)


def pool(lib, d):
    return lib.p100_paged_pool_init(C.byref(d), Z, Z, Z, None)


@pytest.mark.parametrize("kw,why", [
    (dict(n_seq=-1), "counts must not be negative"),
    (dict(n_seq=P.PAGED_MAX_SEQ + 1), "n_seq exceeds P100_PAGED_MAX_SEQ"),
    (dict(page_size=0), "all dimensions must be positive"),
    (dict(head_dim=96), "head_dim must be 64 or 128"),
    (dict(dtype=P.F32), "dtype must be P100_F16 or P100_BF16"),
    (dict(max_pages=1 << 30), "max_pages * page_size exceeds 2^31 - 1"),
    (dict(page_stride=4100), "strides must be multiples of 8 elements"),
])
def test_descriptor_refusals(lib, kw, why):
    d = desc(**kw)
    for call in (plan, pool, append, tree, keep):
        assert call(lib, d) == P.ERR_INVALID
        assert P.last_error() == why


def test_null_descriptor(lib):
    for name, args in (("paged_plan", 10), ("paged_pool_init", 4), ("paged_keep", 9)):
        assert getattr(lib, "p100_" + name)(*[None] * args, None) == P.ERR_INVALID
        assert P.last_error() == "null descriptor"


def test_tree_refusals(lib):
    for words in (0, -1, 33):
        assert tree(lib, desc(), words) == P.ERR_INVALID
        assert P.last_error() == "mask_words must be between 1 and 32"
        assert lib.p100_tree_mask(Z, Z, Z, 1, 1, words, Z, Z, None) == P.ERR_INVALID
        assert P.last_error() == "mask_words must be between 1 and 32"
    for n_seq, n_tokens, why in ((-1, 1, "counts must not be negative"), (1, -1, "counts must not be negative"),
                                 (1025, 1, "n_seq exceeds P100_PAGED_MAX_SEQ")):
        assert lib.p100_tree_mask(Z, Z, Z, n_seq, n_tokens, 1, Z, Z, None) == P.ERR_INVALID
        assert P.last_error() == why


def test_append_refusals(lib):
    d = desc(head_dim=64)
    for kw, why in ((dict(kind=7), "unknown qkv type 7"), (dict(stride=100), "qkv_stride must be at least a fused row"),
                    (dict(stride=12 * 64 + 2), "qkv rows must be 16-byte aligned"),
                    (dict(norm=Z, eps=-1.0), "eps must be finite and non-negative"),
                    (dict(rope=P.Rope(96, 10000.0)), "rope_dim must be at most head_dim")):
        assert append(lib, d, **kw) == P.ERR_INVALID
        assert P.last_error() == why
    for field, value, why in (("rope_dim", 0, "rope_dim must be even and at least 2"),
                              ("rope_dim", 31, "rope_dim must be even and at least 2"),
                              ("mscale", math.nan, "rope's mscale must be finite")):
        rope = P.Rope(64, 10000.0)
        setattr(rope, field, value)
        assert append(lib, d, rope) == P.ERR_INVALID
        assert P.last_error() == why
    assert lib.p100_paged_append_rope(C.byref(d), Z, P.F32, 0, None, None, 0.0, None, *[Z] * 7, None) == P.ERR_INVALID
    assert P.last_error() == "rope must be given"


@pytest.mark.parametrize("kw,why", [
    (dict(rope_dim=0), "rope_dim must be even, between 2 and 128"),
    (dict(rope_dim=33), "rope_dim must be even, between 2 and 128"),
    (dict(rope_dim=130), "rope_dim must be even, between 2 and 128"),
    (dict(theta=0.0), "theta must be positive and finite"),
    (dict(theta=math.nan), "theta must be positive and finite"),
    (dict(scaling=6), "unknown rope scaling"),
    (dict(mscale=-1.0), "mscale must be finite and non-negative"),
    (dict(scaling=P.ROPE_LINEAR), "factor must be positive and finite"),
    (dict(scaling=P.ROPE_NTK, factor=math.inf), "factor must be positive and finite"),
    (dict(scaling=P.ROPE_NTK, factor=2.0, rope_dim=2), "NTK scaling needs rope_dim of at least 4"),
    (dict(scaling=P.ROPE_BANDS, factor=2.0, low=1.0, high=4.0), "original must be positive"),
    (dict(scaling=P.ROPE_BANDS, factor=2.0, low=4.0, high=1.0, original=64), "low and high must be positive, low below high"),
    (dict(scaling=P.ROPE_YARN, factor=2.0, low=1.0, high=math.nan, original=64), "low and high must be positive, low below high"),
    (dict(scaling=P.ROPE_YARN, factor=2.0, low=1.0, high=32.0, original=64, theta=1.0), "YARN scaling needs theta above 1"),
    (dict(scaling=P.ROPE_DIVISORS), "divisors must be given"),
    (dict(scaling=P.ROPE_DIVISORS, rope_dim=4, divisors=[1.0, 0.0]), "divisors must be positive and finite"),
    (dict(theta=1e-30, rope_dim=64), "frequency of pair 18 is too high"),
])
def test_rope_refusals(lib, kw, why):
    with pytest.raises(P.InvalidArgument) as e:
        P.Rope(**{**dict(rope_dim=64, theta=10000.0), **kw})
    assert e.value.message == why


def test_rope_divisors_of_another_length(lib):
    with pytest.raises(P.InvalidArgument):
        P.Rope(8, 10000.0, scaling=P.ROPE_DIVISORS, divisors=[1.0] * 3)


def turns_of(rope):
    return np.array(rope.turns[:rope.rope_dim // 2], dtype=np.longdouble) / np.longdouble(2) ** 64


@pytest.mark.parametrize("rope_dim", [2, 20, 64, 128])
def test_frequencies(lib, rope_dim):
    """Turns a token against the formulas in long double: their own rounding is 2^-65, the formulas' 2^-60 relative."""
    pi2 = 2 * np.longdouble("3.14159265358979323846264338327950288")
    i = np.arange(rope_dim // 2).astype(np.longdouble)
    f = np.longdouble(10000) ** (-2 * i / rope_dim)
    near = lambda rope, want: np.abs(turns_of(rope) - want / pi2) <= 2.0 ** -58 * np.abs(want) + 2.0 ** -64   # noqa: E731
    assert near(P.Rope(rope_dim, 10000.0), f).all()
    assert P.Rope(rope_dim, 10000.0).mscale == 1.0 and not P.Rope(rope_dim, 10000.0).half
    assert near(P.Rope(rope_dim, 10000.0, scaling=P.ROPE_LINEAR, factor=8.0), f / 8).all()
    d = [1.5 + k for k in range(rope_dim // 2)]
    rope = P.Rope(rope_dim, 10000.0, half=True, scaling=P.ROPE_DIVISORS, divisors=d, mscale=1.25)
    assert near(rope, f / np.array(d, np.longdouble)).all() and rope.mscale == 1.25 and rope.half
    if rope_dim > 2:
        g = (np.longdouble(10000) * np.longdouble(4) ** (np.longdouble(rope_dim) / (rope_dim - 2))) ** (-2 * i / rope_dim)
        assert near(P.Rope(rope_dim, 10000.0, scaling=P.ROPE_NTK, factor=4.0), g).all()


def test_bands_and_yarn(lib):
    """The fastest pairs keep their frequency, the slowest are divided, those between lie between and fall."""
    pi2 = 2 * math.pi
    f = 500000.0 ** (-2 * np.arange(64) / 128)
    rope = P.Rope(128, 500000.0, scaling=P.ROPE_BANDS, factor=8.0, low=1.0, high=4.0, original=8192)
    ratio = np.array(turns_of(rope), np.float64) * pi2 / f
    turns = 8192 * f / pi2
    assert np.allclose(ratio[turns >= 4], 1, rtol=1e-12) and np.allclose(ratio[turns <= 1], 1 / 8, rtol=1e-12)
    mid = (turns > 1) & (turns < 4)
    assert mid.sum() > 2 and np.allclose(ratio[mid], 1 / 8 + (turns[mid] - 1) / 3 * 7 / 8, rtol=1e-12)
    rope = P.Rope(128, 10000.0, scaling=P.ROPE_YARN, factor=16.0, low=1.0, high=32.0, original=4096)
    ratio = np.array(turns_of(rope), np.float64) * pi2 / 10000.0 ** (-2 * np.arange(64) / 128)
    lo = math.floor(128 * math.log(4096 / (32 * pi2)) / (2 * math.log(10000)))
    hi = math.ceil(128 * math.log(4096 / pi2) / (2 * math.log(10000)))
    want = 1 - np.clip((np.arange(64) - lo) / (hi - lo), 0, 1) * 15 / 16
    assert np.allclose(ratio, want, rtol=1e-12) and rope.mscale == np.float32(0.1 * math.log(16) + 1)
    assert P.Rope(128, 10000.0, scaling=P.ROPE_YARN, factor=0.5, low=1.0, high=32.0, original=4096).mscale == 1.0


@pytest.mark.skipif(not no_gpu(), reason="checks the behaviour without a GPU")
def test_without_a_device(lib):
    d = desc(head_dim=64)
    for call in (plan, pool, append, tree, keep):
        assert call(lib, d) == P.ERR_UNSUPPORTED
    assert lib.p100_tree_mask(Z, Z, Z, 1, 1, 1, Z, Z, None) == P.ERR_UNSUPPORTED


@pytest.mark.gpu
def test_null_buffers(cuda, lib):
    d = desc(head_dim=64)
    rope = P.Rope(64, 10000.0)
    calls = [
        lambda z: lib.p100_paged_plan(C.byref(d), *z(9, (7, 8)), None),
        lambda z: lib.p100_paged_pool_init(C.byref(d), *z(3), None),
        lambda z: lib.p100_paged_append_rope(C.byref(d), z.one(0), P.F32, 0, None, None, 0.0, C.byref(rope), None,
                                             *z(6, (), 1), None),
        lambda z: lib.p100_paged_keep(C.byref(d), *z(8, (7,)), None),
    ]

    class Args:
        """All given but the `out`-th."""
        def __init__(self, out):
            self.out = out

        def one(self, i):
            return None if i == self.out else Z

        def __call__(self, n, optional=(), first=0):
            return [None if i + first == self.out or i in optional else Z for i in range(n)]

    for call, n in zip(calls, (7, 3, 7, 7)):
        for out in range(n):
            assert call(Args(out)) == P.ERR_INVALID, out
            assert P.last_error() == "null buffer"
    for out in range(8):
        z = [None if i == out else Z for i in range(8)]
        assert lib.p100_fa_tree(C.byref(d), *z[:4], 1, *z[4:8], None, Z, 1 << 40, None) == P.ERR_INVALID
        assert P.last_error() in ("null buffer", "o must not be q")
    for out in (0, 1, 2, 6):
        z = [None if i == out else Z for i in range(7)]
        assert lib.p100_tree_mask(*z[:3], 1, 1, 1, z[6], None, None) == P.ERR_INVALID
        assert P.last_error() == "null buffer"


@pytest.mark.gpu
def test_keep_refuses_shared_arrays(cuda, lib):
    """length may touch none of the arrays that the sequences' blocks read, at either end; refused before any launch."""
    d = desc(head_dim=64)
    at = {name: 4096 * (i + 1) for i, name in enumerate(("k", "v", "keep", "keep_len", "table", "q_start", "kv_len"))}
    ints = {"keep": d.n_tokens, "keep_len": d.n_seq, "table": d.n_seq * d.max_pages, "q_start": d.n_seq + 1, "kv_len": d.n_seq}

    def call(length, **other):
        return lib.p100_paged_keep(C.byref(d), *[C.c_void_p(x) for x in {**at, **other}.values()], C.c_void_p(length), None)

    for name, n in ints.items():
        for length in (at[name], at[name] + 4 * (n - 1), at[name] - 4 * (d.n_seq - 1)):
            assert call(length) == P.ERR_INVALID, name
            assert P.last_error() == "length must not overlap the other arrays"
    assert call(1 << 20, v=at["k"]) == P.ERR_INVALID
    assert P.last_error() == "v_pages must not be k_pages"
