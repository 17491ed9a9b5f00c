"""GPU: hidden sizes at which the logits are summed up chunk by chunk, under the bounds of test_linear_loss_gpu.py."""
import pytest
import torch

from test_linear_loss_gpu import DT, check, head, labels_for, one_hot_args, reference, teacher_args

pytestmark = pytest.mark.gpu

SIZES = [
    # N, D, V, dtype, order, bias: one and several row blocks, single CTAs and pairs, chunks of equal and of unequal length
    (1, 4096, 700, "bf16", "vd", False),
    (20, 2000, 3001, "fp16", "vd", True),
    (128, 1544, 900, "bf16", "dv", True),
    (129, 4096, 777, "bf16", "vd", True),
    (400, 1600, 1032, "fp16", "dv", False),
    (700, 3080, 9001, "bf16", "vd", False),
    (1300, 2304, 20000, "bf16", "dv", True),
    (2600, 5000, 6000, "fp16", "vd", True),
]


@pytest.mark.parametrize("N,D,V,dtype,order,bias", SIZES)
def test_cross_entropy(pkg, cuda, N, D, V, dtype, order, bias):
    gen, x, w, b, g = head(N, D, V, DT[dtype], cuda, order, bias)
    labels = labels_for(gen, N, V, 0.2).to(cuda)
    loss, lse = pkg.linear_cross_entropy(x, w, labels, bias=b)
    grads = pkg.linear_cross_entropy_backward(x, w, labels, lse, g, bias=b)
    check(reference(x, w, b, *one_hot_args(labels, V), 1.0, 1.0, g), DT[dtype], loss, lse, grads)


@pytest.mark.parametrize("N,D,V,dtype,order,bias", SIZES)
def test_distillation(pkg, cuda, N, D, V, dtype, order, bias):
    gen, x, w, b, g = head(N, D, V, DT[dtype], cuda, order, bias)
    K = 30
    index = (torch.randint(0, V, (N, 1), generator=gen) + torch.arange(K) * (V // K - 1)) % V
    index[3:: 9] = -1
    index, logits = index.to(cuda), (torch.randn(N, K, generator=gen) * 3).to(cuda)
    loss, lse = pkg.linear_distillation(x, w, index, logits, bias=b, temperature=2.0)
    grads = pkg.linear_distillation_backward(x, w, index, logits, lse, g, bias=b, temperature=2.0)
    check(reference(x, w, b, *teacher_args(index, logits, 2.0, V), 0.5, 4.0, g), DT[dtype], loss, lse, grads)
