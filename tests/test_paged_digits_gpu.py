"""How many digits p100_fa_paged keeps of the probabilities, with fp32 outputs against 64 bits.

Bound of o: (rel + 2 e + 2^-18) sum p |v| + tail sum |v| + 2^-24 with e, 2^-18 and 2^-24 as in test_paged_gpu.py, `rel`
what is lost of a probability relative to it, `tail` what a small one loses of the row's largest.

Single tokens carry a probability in two 16-bit parts, each rounded to nearest: rel = u^2 (2^-16 in bfloat16, 2^-22 in
float16).  In float16 the largest is 2^15 and nothing below 2^-25 is held, so tail = 2^-40; bfloat16 has FP32's range.
Chunks round a probability once, rel = u; in float16 the largest is 2^7 or more, so tail = 2^-32."""
import math

import pytest

from test_paged_gpu import Batch, attend

import p100_b200 as P

pytestmark = pytest.mark.gpu


def check64(torch, b, q, o, rel, tail, causal=True):
    group, scale = b.hq // b.hkv, 1.0 / math.sqrt(b.dim)
    for s, (n, t) in enumerate(zip(b.q_lens, b.kv_lens)):
        lo = int(b.q_start_host[s])
        k, v = b.rows(b.k, s), b.rows(b.v, s)
        seen = torch.arange(t, device="cuda")[None] < (t - n + 1 + torch.arange(n, device="cuda"))[:, None]
        for h in range(b.hq):
            qh, kh, vh = q[lo:lo + n, h].double(), k[:, h // group], v[:, h // group]
            x = qh @ kh.T * scale
            e = b.dim * 2.0 ** -24 * scale * (qh.abs() @ kh.abs().T) + 2.0 ** -20
            if causal:
                x, e = x.masked_fill(~seen, -math.inf), e.masked_fill(~seen, 0.0)
            p = torch.softmax(x, 1)
            tol = (rel + 2 * e.amax(1, keepdim=True) + 2.0 ** -18) * (p @ vh.abs()) + tail * vh.abs().sum(0) + 2.0 ** -24
            d = (o[lo:lo + n, h].double() - p @ vh).abs()
            assert bool((d <= tol).all()), f"sequence {s}, head {h}: off by {float((d / tol).max()):.3g} of the bound"


def kept(torch, b):
    u = torch.finfo(b.t).eps / 2
    return u * u, 2.0 ** -40 if b.t == torch.float16 else 0.0


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,dim", [(8, 1, 128), (8, 8, 64), (12, 1, 128), (15, 1, 64), (32, 2, 128)])
@pytest.mark.parametrize("lens", [[5, 700, 64, 1], [3000]])
def test_digits_of_single_tokens(cuda, lens, hq, hkv, dim, dtype):
    """At most 8 rows of a kv head, whose rests lie beside them, and up to 16, whose rests take products of their own."""
    b = Batch(cuda, [1] * len(lens), lens, hq, hkv, dim, dtype, 16, seed=70)
    b.fill()
    q = b.queries(3.0)
    o, _ = attend(b, q, o_fp32=True)
    check64(cuda, b, q, o, *kept(cuda, b))


def far_tail(torch, q_lens, kv_len, dtype):
    """One key far above all others, whose value is 0: what a row gives is the sum of probabilities of e^-17.5 each
    (2^-25.2), a thousandth together."""
    b = Batch(torch, q_lens, [kv_len] * len(q_lens), 4, 1, 64, dtype, 64, seed=71)
    for s in range(len(q_lens)):
        page, off = b.slots(s)
        b.k[page, :, off] = -35 / 16   # 64 products over sqrt(64)
        b.v[page, :, off] = 1.0
        b.k[page[0], :, off[0]] = b.v[page[0], :, off[0]] = 0.0
    return b, torch.ones(b.n_tokens, b.hq, b.dim, dtype=b.t, device="cuda")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("group", [4, 12])
def test_far_tails_of_single_tokens(cuda, dtype, group):
    b, q = far_tail(cuda, [1, 1], 65536, dtype)
    b.hq = group
    q = q[:, :1].expand(-1, group, -1).contiguous()
    o, _ = attend(b, q, o_fp32=True)
    assert 1e-3 < float(o.min()) and float(o.max()) < 2e-3
    check64(cuda, b, q, o, *kept(cuda, b))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_far_tails_of_chunks(cuda, dtype):
    b, q = far_tail(cuda, [40, 9], 65536, dtype)
    o, _ = attend(b, q, o_fp32=True)
    assert 1e-3 < float(o.min()) and float(o.max()) < 2e-3
    check64(cuda, b, q, o, cuda.finfo(b.t).eps / 2, 2.0 ** -32 if dtype == "f16" else 0.0)
