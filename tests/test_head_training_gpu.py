"""GPU: the end of a training step through the kernels against autograd on the same numbers in 64 bits.

The hidden states after the norm, their gradient and the results are rounded to 16 bits on the way (u = 2^-8 bf16, 2^-11 fp16
each): the rounded norm output moves a logit by up to u |h| |w| and the loss and every gradient with it, so results are held to
8 u of their own size (2-norm), the loss to 4 u."""
import importlib

import pytest
import torch

from test_head_training_cpu import case, expected, targets

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind,bias", [("rms", False), ("layer", True)])
@pytest.mark.parametrize("distill", [False, True])
def test_kernel_pass_against_autograd(pkg, cuda, dtype, kind, bias, distill):
    layers = importlib.import_module(pkg.__name__ + ".layers")
    g, x, w = case(layers, kind, bias, seed=4, dtype=dtype)
    labels, teacher = targets(g, distill)
    T = 2.0 if distill else 1.0
    want, wanted = expected(x, w, labels, teacher, T, 64.0)
    put = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    on_gpu = layers.LmHeadWeights(weight=put(w.weight), gain=put(w.gain), kind=kind, shift=put(w.shift), bias=put(w.bias), eps=w.eps)
    before = pkg.launch_count()
    loss, grads = layers.lm_head_training_pass(put(x), on_gpu, layers.KernelOps(pkg), labels=put(labels),
                                               teacher=None if teacher is None else tuple(put(t) for t in teacher), temperature=T,
                                               loss_scale=64.0)
    assert pkg.launch_count() > before
    assert abs(loss.item() - want.item()) <= 4 * U[dtype] * abs(want.item())
    for name, ref in wanted.items():
        got = getattr(grads, name)
        assert got.dtype == dtype
        assert (got.double().cpu() - ref).norm() <= 8 * U[dtype] * ref.norm(), name


def test_no_synchronisation(pkg, cuda):
    """A pass can be captured in a CUDA graph, which a wait for the GPU would break, and replays to the same bits."""
    layers = importlib.import_module(pkg.__name__ + ".layers")
    g, x, w = case(layers, "rms", False, dtype=torch.bfloat16)
    labels = targets(g, False)[0].to(cuda)
    x = x.to(cuda)
    w = layers.LmHeadWeights(weight=w.weight.to(cuda), gain=w.gain.to(cuda))
    ops = layers.KernelOps(pkg)
    loss, grads = layers.lm_head_training_pass(x, w, ops, labels=labels)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            loss2, grads2 = layers.lm_head_training_pass(x, w, ops, labels=labels)
        graph.replay()
    stream.synchronize()
    assert torch.equal(loss, loss2) and torch.equal(grads.x, grads2.x) and torch.equal(grads.weight, grads2.weight)
