"""GPU: infinities in norm and rotation of heads stay where the formula has them: columns that do not turn depend on no other
column's product, and columns that turn on their pair's alone."""
import math

import pytest
import torch

from test_qk_norm_rotary_gpu import angles, inputs

pytestmark = pytest.mark.gpu


def pair_of(column, rotary, half):
    if column >= rotary:
        return {column}
    if half:
        return {column, (column + rotary // 2) % rotary}
    return {column, column ^ 1}


SIZES = [(64, 16), (128, 32), (128, 64), (256, 64), (80, 32), (40, 16)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("H,rotary", SIZES)
def test_forward(pkg, cuda, dtype, half, H, rotary):
    """A head with an infinity has r = 0: its numbers become 0, the infinity's own column NaN, and its pair's where it turns."""
    columns = sorted({0, rotary // 2, rotary - 1, rotary, rotary + 5, H // 2 + rotary // 2, H - 1} & set(range(H)))
    T, N, NK = len(columns), 3, 2
    s = inputs(cuda, T, N, NK, H, dtype, dtype, rotary, seed=H)
    for t, column in enumerate(columns):
        s["q"][t, 1, column] = math.inf
        s["k"][t, 1, column] = -math.inf
    q, k = pkg.qk_norm_rotary_forward(s["q"], s["k"], q_gain=s["q_gain"], k_gain=s["k_gain"], cos=s["cos"], sin=s["sin"],
                                      positions=s["positions"], half_split=half)
    for y in (q, k):
        for t, column in enumerate(columns):
            odd = torch.zeros(H, dtype=torch.bool, device=cuda)
            odd[list(pair_of(column, rotary, half))] = True
            assert (y[t, 1][~odd] == 0).all(), (column, y[t, 1].isnan().nonzero()[:, 0].tolist())
            assert y[t, 1, column].isnan() and y[t, 0].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("H,rotary", SIZES)
def test_gains(pkg, cuda, dtype, half, H, rotary):
    """An infinite gain of a column that does not turn stays in that column."""
    s = inputs(cuda, 40, 3, 2, H, dtype, dtype, rotary, seed=H)
    s["q_gain"][rotary + 3] = math.inf
    q, k = pkg.qk_norm_rotary_forward(s["q"], s["k"], q_gain=s["q_gain"], k_gain=s["k_gain"], cos=s["cos"], sin=s["sin"],
                                      positions=s["positions"], half_split=half)
    odd = torch.zeros(H, dtype=torch.bool, device=cuda)
    odd[rotary + 3] = True
    assert q[..., ~odd].isfinite().all() and k.isfinite().all()
    x = s["q"][..., rotary + 3]
    assert torch.equal(q[..., rotary + 3][x != 0], (x.sign() * math.inf)[x != 0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("H,rotary", SIZES)
def test_backward(pkg, cuda, dtype, half, H, rotary):
    """An infinite gradient of a column that does not turn: its own gain's gradient, and no other column's."""
    for column in sorted({rotary, rotary + 5, H // 2 + rotary // 2, H - 1} & set(range(rotary, H))):
        s = inputs(cuda, 50, 3, 2, H, dtype, dtype, rotary, seed=H)
        s["grad_q"][7, 2, column] = math.inf
        dq, dk, dqg, dkg = pkg.qk_norm_rotary_backward(s["grad_q"], s["grad_k"], s["q"], s["k"], q_gain=s["q_gain"], k_gain=s["k_gain"],
                                                       cos=s["cos"], sin=s["sin"], positions=s["positions"], half_split=half)
        odd = torch.zeros(H, dtype=torch.bool, device=cuda)
        odd[column] = True
        assert dqg[~odd].isfinite().all(), (column, (~dqg.isfinite()).nonzero()[:, 0].tolist())
        assert dqg[column] == math.inf * s["q"][7, 2, column].sign() and dkg.isfinite().all() and dk.isfinite().all()
        there = torch.ones_like(dq[..., 0], dtype=torch.bool)
        there[7, 2] = False
        assert dq[there].isfinite().all()
    assert angles(s, 50)[0].isfinite().all()
