"""GPU: the end of a training step whose head has a bias and whose vocabulary is taken in several pieces, against autograd on the same
numbers in 64 bits, under the bounds of test_head_training_gpu.py, the first rows of the hidden states' gradient by themselves too."""
import importlib

import pytest
import torch

from test_head_training_cpu import expected

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("distill", [False, True])
@pytest.mark.parametrize("tokens,vocab", [(8192, 50400), (16384, 17000)])
def test_kernel_pass_against_autograd(pkg, cuda, distill, tokens, vocab):
    layers = importlib.import_module(pkg.__name__ + ".layers")
    gen = torch.Generator(device=cuda).manual_seed(tokens)
    r = lambda *s: torch.randn(*s, generator=gen, device=cuda).bfloat16()  # noqa: E731
    w = layers.LmHeadWeights(weight=r(vocab, 64) * 0.2, gain=r(64) * 0.1 + 1, kind="layer", shift=r(64) * 0.1, bias=r(vocab) * 0.3, eps=1e-5)
    x = r(4, tokens // 4, 64)
    labels = torch.randint(0, vocab, (4, tokens // 4), generator=gen, device=cuda)
    labels[0, :70] = -100
    index = (labels[..., None] + torch.arange(6, device=cuda) * 1000) % vocab
    index[0, :70] = -1
    labels, teacher, T = (None, (index, r(4, tokens // 4, 6) * 2), 2.0) if distill else (labels, None, 1.0)
    want, wanted = expected(x, w, labels, teacher, T, 64.0)
    loss, grads = layers.lm_head_training_pass(x, w, layers.KernelOps(pkg), labels=labels, teacher=teacher, temperature=T, loss_scale=64.0)
    u = 2.0 ** -8
    assert abs(loss.item() - want.item()) <= 4 * u * abs(want.item())
    for name, ref in wanted.items():
        assert (getattr(grads, name).double() - ref).norm() <= 8 * u * ref.norm(), name
    assert (grads.x[0, :70] == 0).all()
    first, ref = grads.x[0, 70:90].double(), wanted["x"][0, 70:90]
    assert ((first - ref).norm(dim=1) <= 8 * u * ref.norm(dim=1)).all()
