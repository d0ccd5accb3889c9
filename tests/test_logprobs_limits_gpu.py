"""p100_logprobs at the largest number of logits that it takes, in rows that are not split."""
import math

import pytest

import p100_b200 as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_ranks_of_the_longest_rows(cuda, dtype):
    """2^24 equal (or masked) 16-bit logits, so many rows that each is one block's: a thread counts 2^16 of them in each
    half of its packed words.  Rank and alternatives follow the index; ln of the number of logits is known."""
    torch = cuda
    n, rows = 1 << 24, 600
    x = torch.zeros((rows, n), dtype=getattr(torch, dtype), device="cuda")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    tokens = torch.randint(0, n, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    tokens[:4] = torch.tensor([n - 1, 0, n - 8, n - 9], dtype=torch.int32)
    masked = rows - 3
    x[masked:] = -math.inf
    x[masked:, 3] = 1.0   # the only real logit of the last rows; rank counts the masked ones in front of a masked token
    tokens[masked:] = torch.tensor([n - 1, 3, n - 4096], dtype=torch.int32)
    r = P.logprobs(x, tokens, top_k=1)
    P.check(P.device_error())
    want = tokens.clone()
    want[masked + 1] = 0
    assert torch.equal(r.rank, want)
    assert torch.equal(r.top_index[:masked, 0], torch.zeros_like(want[:masked]))
    assert torch.equal(r.top_index[masked:, 0], torch.full_like(want[masked:], 3))
    # equal logits: every exponential is 1 and every sum a whole number below 2^24 (or 2^24 itself); ln is within 2^-22 of it
    assert bool(((r.entropy[:masked] - math.log(n)).abs() <= 2.0 ** -22 * math.log(n)).all())
    assert bool(((r.logprob[:masked] + math.log(n)).abs() <= 2.0 ** -22 * math.log(n)).all())
    assert bool((r.entropy[masked:] == 0).all()) and float(r.logprob[masked + 1]) == 0.0
    assert bool(torch.isneginf(r.logprob[[masked, masked + 2]]).all())
