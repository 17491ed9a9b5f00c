"""GPU: teacher logits as large as their type allows, at temperatures below 1, under the bounds of test_linear_loss_gpu.py (the
teacher's softmax is of differences of logits, which the temperature may take beyond fp32 without harm: those entries weigh 0)."""
import pytest
import torch

from test_linear_loss_gpu import check, head, reference, teacher_args

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("teacher", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [60, 300])
def test_logits_at_the_ends_of_the_type(pkg, cuda, teacher, N):
    V, K, T = 500, 6, 0.25
    gen, x, w, b, g = head(N, 64, V, torch.bfloat16, cuda, bias=True)
    x = x * 0.25      # (logits over T about as usual)
    index = torch.stack([torch.randperm(V, generator=gen)[:K] for _ in range(N)]).to(cuda)
    logits = torch.randn(N, K, generator=gen).to(cuda).to(teacher)
    lowest, largest = torch.finfo(teacher).min, torch.finfo(teacher).max
    logits[0::5] = lowest                 # all masked by the lowest number: the entries are there, and alike
    logits[1::5, 2:] = lowest             # some of them
    logits[2::5, 0] = largest             # one above all
    logits[3::5, :3] = largest
    loss, lse = pkg.linear_distillation(x, w, index, logits, bias=b, temperature=T)
    grads = pkg.linear_distillation_backward(x, w, index, logits, lse, g, bias=b, temperature=T)
    check(reference(x, w, b, *teacher_args(index, logits, T, V), 1 / T, T * T, g), torch.bfloat16, loss, lse, grads)
