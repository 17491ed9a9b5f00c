"""GPU: paged attention of stretches of new tokens of many tiles without a mask, against the definition in 64 bits (tolerance: see
test_fmha_paged_gpu).  Units whose keys all rows of a tile see, those that end in the tile's own tokens, and those with both;
tiles of whole and of few rows; stale keys and values behind the last token (NaN), and infinite ones before it."""
import math

import pytest
import torch

from test_fmha_paged_gpu import call, check, make

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
CASES = [
    # lengths, new tokens, heads, kv heads, head size, page, type
    ([0], [1500], 4, 2, 128, 16, BF),
    ([37, 700], [1100, 129], 8, 2, 64, 64, HF),
    ([63, 64, 65], [129, 128, 127], 4, 4, 128, 8, BF),         # tiles of 128 tokens
    ([5], [900], 16, 1, 128, 32, BF),                          # tiles of 8 tokens: most units are seen whole
    ([1000, 0, 3], [200, 1, 333], 67, 1, 80, 16, HF),          # of one token
    ([250], [700], 6, 2, 256, 16, HF),
    ([31], [513], 5, 1, 192, 8, BF),
    ([0, 10, 20, 30], [64, 65, 63, 300], 12, 4, 128, 256, BF),
    ([100] * 40, [70] * 40, 8, 8, 64, 16, BF),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"L{c[0][0]}x{len(c[0])}n{c[1][0]}N{c[2]}K{c[3]}H{c[4]}P{c[5]}{str(c[6])[6:]}")
def test_against_the_definition(pkg, cuda, case):
    lengths, new, heads, kv, size, page, dtype = case
    s = make(cuda, lengths, new, heads, kv, size, page, dtype, seed=sum(new))
    out, lse = call(pkg, s)
    check(s, out, lse)
    # the first rows alone, as a shorter stretch of the same tokens, are the same to a rounding of the split over workers
    if len(new) == 1:
        n = new[0] // 3
        t = dict(s, q=s["q"][:n], granted=s["granted"].clone().fill_(n), row_start=torch.tensor([0, n], dtype=torch.int32, device=cuda))
        check(t, *call(pkg, t))


def test_a_table_that_ends_inside_the_stretch(pkg, cuda):
    """Tokens without a place in the table are not read, and do not make others visible."""
    s = make(cuda, [50], [400], 4, 2, 128, 8, BF)
    whole, whole_lse = call(pkg, s)
    cut = 40 * 8
    t = dict(s, table=s["table"][:, :40].contiguous())
    out, lse = call(pkg, t)
    n = cut - 50          # rows whose own token is in the table
    # (the runs differ, and with them where parts are joined)
    assert torch.allclose(out[:n].float(), whole[:n].float(), atol=0.03, rtol=0.02) and torch.allclose(lse[:n], whole_lse[:n], atol=1e-3)
    k = s["k"][t["table"][0].long()].flatten(0, 1).double().repeat_interleave(2, 1).transpose(0, 1)
    z = s["q"][n:].double().transpose(0, 1) @ k.transpose(1, 2) * s["scale"]
    assert torch.allclose(lse[n:].double(), torch.logsumexp(z, 2).t(), atol=1e-3) and out.isfinite().all()


def test_infinite_values_before_a_tile(pkg, cuda):
    """An infinite value of an early token is that value in all later rows and in no earlier one."""
    s = make(cuda, [20], [600], 4, 2, 128, 16, BF, seed=9)
    want, _ = call(pkg, s)
    t = 20 + 100
    s["v"][s["table"][0, t // 16].long(), t % 16, 1, 7] = -math.inf
    out, _ = call(pkg, s)
    assert (out[100:, 2:, 7] == -math.inf).all() and out[:100].isfinite().all()
    out[100:, 2:, 7] = want[100:, 2:, 7]
    assert torch.equal(out, want)
