"""p100_fa_paged at the ends of what its descriptor takes, with the bounds of test_paged_gpu.py."""
import pytest

from test_paged_gpu import Batch, attend, attend64, check

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
