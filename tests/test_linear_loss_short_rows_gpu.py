"""GPU: hidden sizes below one 16-byte vector, with gradients whose rows are apart by whole vectors, under the bounds of
test_linear_loss_gpu.py."""
import pytest
import torch

from test_linear_loss_gpu import check, head, labels_for, one_hot_args, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N", [100, 300])
@pytest.mark.parametrize("D,order", [(4, "vd"), (7, "dv"), (1, "vd")])
def test_hidden_sizes_below_a_vector(pkg, cuda, N, D, order):
    gen, x, w, b, g = head(N, D, 50, torch.bfloat16, cuda, order, bias=True)
    labels = labels_for(gen, N, 50, 0.2).to(cuda)
    loss, lse = pkg.linear_cross_entropy(x, w, labels, bias=b)
    wide = torch.full((N, 16), 5.0, dtype=x.dtype, device=cuda)
    grads = pkg.linear_cross_entropy_backward(x, w, labels, lse, g, bias=b, grad_x=wide[:, :D])
    assert (wide[:, D:] == 5).all()
    check(reference(x, w, b, *one_hot_args(labels, 50), 1.0, 1.0, g), torch.bfloat16, loss, lse, grads)
    dense = pkg.linear_cross_entropy_backward(x, w, labels, lse, g, bias=b)
    for a, c in zip(grads, dense):
        assert torch.equal(a, c)
