"""GPU: row counts at which one CTA of the gather has more rows than threads."""
import pytest
import torch

from test_linear_loss_gpu import check, head, labels_for, one_hot_args, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N", [262145, 600001])
def test_against_64_bits(pkg, cuda, N):
    """The bounds of test_linear_loss_gpu.py."""
    gen, x, w, b, g = head(N, 8, 24, torch.bfloat16, cuda, bias=True)
    labels = labels_for(gen, N, 24, 0.4).to(cuda)
    loss, lse = pkg.linear_cross_entropy(x, w, labels, bias=b)
    grads = pkg.linear_cross_entropy_backward(x, w, labels, lse, g, bias=b)
    check(reference(x, w, b, *one_hot_args(labels, 24), 1.0, 1.0, g), torch.bfloat16, loss, lse, grads)


def test_time_grows_with_the_rows(pkg, cuda):
    """Eight times the rows take eight times as long (and at most twice that), not 64 times."""
    w = torch.randn(16, 8, device=cuda).bfloat16()
    times = []
    for N in (1 << 20, 1 << 23):
        x = torch.randn(N, 8, device=cuda, dtype=torch.bfloat16)
        labels = torch.randint(0, 16, (N,), device=cuda)
        ws = torch.empty(pkg.linear_loss_workspace_bytes(x, w), dtype=torch.uint8, device=cuda)
        best = float("inf")
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            pkg.linear_cross_entropy(x, w, labels, workspace=ws)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        times.append(best)
    assert times[1] <= 16 * times[0], times
