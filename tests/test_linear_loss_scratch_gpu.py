"""GPU: calls at the vocabulary head with exactly the scratch that the query tells, whatever the weight's layout."""
import pytest
import torch

from test_linear_loss_gpu import head, labels_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("order", ["vd", "dv"])
@pytest.mark.parametrize("N", [128, 129])
def test_queried_scratch_is_enough(pkg, cuda, order, N):
    gen, x, w, b, g = head(N, 64, 1000, torch.bfloat16, cuda, order, bias=True)
    labels = labels_for(gen, N, 1000, 0.2).to(cuda)
    index, logits = torch.randint(0, 1000, (N, 5), generator=gen).to(cuda), torch.randn(N, 5, generator=gen).to(cuda)

    def scratch(entries, backward):
        return torch.empty(pkg.linear_loss_workspace_bytes(x, w, entries, backward), dtype=torch.uint8, device=cuda)

    for entries, forward, back in (
            (0, lambda **kw: pkg.linear_cross_entropy(x, w, labels, bias=b, **kw),
             lambda lse, **kw: pkg.linear_cross_entropy_backward(x, w, labels, lse, g, bias=b, **kw)),
            (5, lambda **kw: pkg.linear_distillation(x, w, index, logits, bias=b, **kw),
             lambda lse, **kw: pkg.linear_distillation_backward(x, w, index, logits, lse, g, bias=b, **kw))):
        loss, lse = forward()
        grads = back(lse)
        again = forward(workspace=scratch(entries, False))
        assert torch.equal(loss, again[0]) and torch.equal(lse, again[1])
        for a, c in zip(grads, back(lse, workspace=scratch(entries, True))):
            assert torch.equal(a, c)
