"""GPU: paged attention of long stretches of new tokens of which some have values that are no numbers.  They reach the rows that see
them, and only those, and cost what they cost, not a walk over all tokens of the stretch."""
import math

import pytest
import torch

from test_fmha_paged_gpu import call, make, random_mask

pytestmark = pytest.mark.gpu


def hurt(s, b, places):
    """Values of request b's new tokens d made no numbers: {d: (key head, column, value)}.  Returns the inputs as they were."""
    clean = dict(s, v=s["v"].clone())
    page, L = s["k"].shape[1], int(s["lengths"][b])
    for d, (head, column, value) in places.items():
        s["v"][s["table"][b, (L + d) // page].long(), (L + d) % page, head, column] = value
    return clean


def odd_for(s, b, places):
    """[n, heads, size]: where a row's result cannot be a number."""
    n, r0 = int(s["granted"][b]), int(s["row_start"][b])
    group = s["q"].shape[1] // s["k"].shape[2]
    odd = torch.zeros(n, *s["q"].shape[1:], dtype=torch.bool, device=s["q"].device)
    for d, (head, column, _) in places.items():
        if s["mask"] is None:
            sees = torch.arange(n, device=odd.device) >= d
        elif d < 32 * s["mask"].shape[1]:
            sees = (s["mask"][r0:r0 + n, d // 32].long() >> (d % 32) & 1) > 0
        else:
            continue
        odd[:, head * group:(head + 1) * group, column] |= sees[:, None]
    return odd


# (requests beside the hurt one, its tokens, its mask's words; heads, kv heads, head size, page, type)
CASES = [
    ([37, 500], [700, 3], 0, 4, 2, 128, 16, torch.bfloat16),
    ([0, 90], [1300, 40], 0, 8, 1, 64, 64, torch.float16),
    ([130, 3], [400, 1], 0, 6, 2, 256, 8, torch.bfloat16),
    ([5, 0], [520, 2], 16, 4, 2, 128, 32, torch.float16),
    ([61, 10], [300, 9], 7, 3, 1, 80, 16, torch.bfloat16),       # tokens behind the mask's last word
    ([20], [2500], 0, 2, 1, 192, 16, torch.bfloat16),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"L{c[0][0]}n{c[1][0]}w{c[2]}N{c[3]}H{c[5]}P{c[6]}")
@pytest.mark.parametrize("many", [False, True])
def test_they_reach_the_rows_that_see_them(pkg, cuda, case, many):
    lengths, new, words, heads, kv, size, page, dtype = case
    s = make(cuda, lengths, new, heads, kv, size, page, dtype, seed=11)
    if words:
        s["mask"] = random_mask(s, words)
    n = new[0]
    values = (math.nan, math.inf, -math.inf)
    places = {d: (d % kv, (7 * d) % size, values[d % 3]) for d in (range(0, n, 3) if many else (0, 5, 63, 64, 65, 200, n - 2, n - 1))}
    clean = hurt(s, 0, places)
    want, want_lse = call(pkg, clean)
    out, lse = call(pkg, s)
    odd = odd_for(s, 0, places)
    assert torch.equal(lse, want_lse)
    assert torch.equal(out[:n].isfinite(), ~odd)
    assert torch.equal(out[:n][~odd], want[:n][~odd]) and torch.equal(out[n:], want[n:])
    again, _ = call(pkg, s)
    assert torch.equal(again.nan_to_num(), out.nan_to_num())
    # a column that one row alone of the values reaches is that value
    for d, (head, column, value) in places.items():
        if many or not math.isinf(value):
            continue
        if any(e != d and places[e][:2] == (head, column) for e in places):
            continue
        group = heads // kv
        x = out[:n, head * group:(head + 1) * group, column]
        sees = odd[:, head * group:(head + 1) * group, column]
        assert (x[sees] == value).all()


def test_parts_of_one_long_stretch(pkg, cuda):
    """One prompt that many workers share."""
    s = make(cuda, [9000], [64], 2, 1, 128, 64, torch.bfloat16, seed=2)
    places = {3: (0, 1, math.inf), 40: (0, 127, math.nan)}
    clean = hurt(s, 0, places)
    (want, _), (out, _) = call(pkg, clean), call(pkg, s)
    odd = odd_for(s, 0, places)
    assert torch.equal(out.isfinite(), ~odd) and torch.equal(out[~odd], want[~odd]) and (out[3:, :, 1] == math.inf).all()


def test_their_cost(pkg, cuda):
    """A prompt of 8192 tokens with one NaN in its first tokens takes about as long as without (a walk over all tokens of the
    prompt for every row behind the NaN made it 400 times as long), and one of nothing else stays far from the limit on waits."""
    s = make(cuda, [0], [8192], 16, 4, 128, 64, torch.bfloat16, seed=3)
    clean = hurt(s, 0, {3: (h, 5, math.nan) for h in range(4)})

    def time(t):
        call(pkg, t)
        best = math.inf
        for _ in range(3):
            e = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            e[0].record()
            call(pkg, t)
            e[1].record()
            e[1].synchronize()
            best = min(best, e[0].elapsed_time(e[1]))
        return best

    usual = time(clean)
    assert time(s) < 3 * usual
    clean["v"].fill_(math.nan)
    assert time(clean) < 40 * usual and call(pkg, clean)[0].isnan().all()
    assert pkg.device_status() == 0
