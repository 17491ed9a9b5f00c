"""GPU: backward passes at the vocabulary head that take the vocabulary in several pieces, against the definitions in 64 bits.

The bounds are those of test_linear_loss_gpu.py.  They hold for any number of pieces: dx is one fp32 sum over the vocabulary, cut
where a piece ends; dw and db of a column come from one piece.  An lse of 600000
columns is a sum whose terms pass through at most 64 additions and 40 changes of the maximum one after the other, 2^-24 and 2^-23
each: 9e-6 of the sum, which 2^-20 (1 + |lse|) holds where the lse is above 12."""
import pytest
import torch

from test_linear_loss_gpu import DT, check, head, labels_for, one_hot_args, reference, teacher_args

pytestmark = pytest.mark.gpu

SIZES = [
    # N, D, V, dtype, order, bias: pieces and the last one's columns
    (16384, 64, 17000, "bf16", "vd", True),      # 5888, 5888, 5224
    (8192, 64, 50400, "bf16", "dv", True),       # 3 x 12800, 12000
    (5274, 32, 37914, "fp16", "vd", True),       # 19200, 18714
    (8192, 40, 50257, "bf16", "vd", False),
    (64, 32, 600000, "bf16", "vd", True),        # one row block: dx is added up by the GEMM for few rows
    (3, 24, 530001, "fp16", "vd", False),
]


@pytest.mark.parametrize("N,D,V,dtype,order,bias", SIZES)
def test_cross_entropy(pkg, cuda, N, D, V, dtype, order, bias):
    gen, x, w, b, g = head(N, D, V, DT[dtype], cuda, order, bias)
    labels = labels_for(gen, N, V, 0.1).to(cuda)
    loss, lse = pkg.linear_cross_entropy(x, w, labels, bias=b)
    grads = pkg.linear_cross_entropy_backward(x, w, labels, lse, g, bias=b)
    check(reference(x, w, b, *one_hot_args(labels, V), 1.0, 1.0, g), DT[dtype], loss, lse, grads)


@pytest.mark.parametrize("N,D,V,dtype,order,bias", [SIZES[0], SIZES[1], SIZES[4]])
def test_distillation(pkg, cuda, N, D, V, dtype, order, bias):
    gen, x, w, b, g = head(N, D, V, DT[dtype], cuda, order, bias)
    K = 12
    index = (torch.randint(0, V, (N, 1), generator=gen) + torch.arange(K) * (V // K - 1)) % V
    index[:: 7] = -1
    index, logits = index.to(cuda), (torch.randn(N, K, generator=gen) * 3).to(cuda)
    loss, lse = pkg.linear_distillation(x, w, index, logits, bias=b, temperature=2.0)
    grads = pkg.linear_distillation_backward(x, w, index, logits, lse, g, bias=b, temperature=2.0)
    check(reference(x, w, b, *teacher_args(index, logits, 2.0, V), 0.5, 4.0, g), DT[dtype], loss, lse, grads)
