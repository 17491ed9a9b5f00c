"""GPU: paged attention whose weights are one large one and a long flat tail of small ones, against the definition in 64 bits.

Tolerance: that of test_fmha_paged_gpu, and a term for weights that are no normal numbers of the type.  The largest weight of a
row is 2^11 or more as an fp16 operand, fp16's subnormal numbers lie 2^-24 apart, so a weight is off by at most 2^-25 / 2^11 =
2^-36 of the largest (which is at most 1 of the sum), on top of the relative rounding: T 2^-36 max |v| for T keys, twice, since the
sum of the rounded weights is off by as much.  (bf16 has fp32's exponents: none.)"""
import math

import pytest
import torch

from test_fmha_paged_gpu import call, expected, make

pytestmark = pytest.mark.gpu


def with_tail(cuda, lengths, new, dtype, where, low, high, size=64, heads=4, kv_heads=2):
    """One key of weight 1 at `where` (a share of the keys) with value 0, all others of 2^-high to 2^-low of it with values 0.5 to 1.5."""
    s = make(cuda, lengths, new, heads, kv_heads, size, 64, dtype, seed=int(high))
    g = torch.Generator(device=cuda).manual_seed(7)
    s["scale"] = 1.0
    s["q"] = torch.zeros_like(s["q"])
    s["q"][..., 0] = 8.0
    s["k"].zero_()
    drop = low + (high - low) * torch.rand(s["k"].shape[:-1], generator=g, device=cuda)
    s["k"][..., 0] = (2.0 - drop * math.log(2.0) / 8.0).to(dtype)
    s["v"].copy_(0.5 + torch.rand(s["v"].shape, generator=g, device=cuda))
    for b, (n, m) in enumerate(zip(lengths, new)):
        t = min(int(where * (n + m)), n + m - 1)
        s["k"][s["table"][b, t // 64].long(), t % 64, :, 0] = 2.0
        s["v"][s["table"][b, t // 64].long(), t % 64] = 0.0
    return s


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("low,high", [(20, 25), (25, 25), (24.6, 24.6), (20, 34)])
@pytest.mark.parametrize("lengths,new,where", [([20000], [1], 0.0), ([65000], [2], 0.5), ([65000], [1], 1.0), ([2000] * 150, [1] * 150, 0.0),
                                               ([2000] * 150, [3] * 150, 0.7)])
def test_small_weights_add_up(pkg, cuda, dtype, low, high, lengths, new, where):
    s = with_tail(cuda, lengths, new, dtype, where, low, high)
    out, lse = call(pkg, s)
    for r0, o, e, tol, tol_lse in expected(s):
        n = o.shape[0]
        keys = max(lengths) + max(new)
        tail = 2 * keys * 2.0 ** -36 * 1.5 if dtype == torch.float16 else 0.0
        off = (out[r0:r0 + n].double() - o).abs()
        assert (off <= tol + tail).all(), f"row {r0}: {(off / (tol + tail)).max():.2f} of the tolerance, {off.max():.3e} of {o.abs().max():.3e}"
        assert ((lse[r0:r0 + n].double() - e).abs() <= tol_lse).all()


def test_a_maximum_that_climbs(pkg, cuda):
    """Every unit's largest score a little above the one before it, by less and by more than what makes the kernel raise its
    reference point: the weights stay inside the type's range."""
    for step in (1.0, 3.9, 4.1, 7.9, 12.0):
        s = with_tail(cuda, [1500], [1], torch.float16, 0.0, 20, 20)
        t = torch.arange(1501, device=cuda)
        climb = (-20.0 + (t // 64) * step / 8.0 * math.log(2.0)).half()
        s["k"][s["table"][0, t // 64].long(), t % 64, :, 0] = climb[:, None]
        s["v"][s["table"][0, t // 64].long(), t % 64] = torch.where(t % 2 == 0, 60000.0, -60000.0).half()[:, None, None]
        out, lse = call(pkg, s)
        for r0, o, e, tol, tol_lse in expected(s):
            off = (out[r0:r0 + 1].double() - o).abs()
            assert (off <= tol + 2 * 1501 * 2.0 ** -36 * 60000.0).all(), (step, (off / tol).max())
            assert ((lse[r0:r0 + 1].double() - e).abs() <= tol_lse).all()
