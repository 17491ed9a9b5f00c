"""CPU: the end of a training step (layers.lm_head_training_pass) in its plain form against autograd in 64 bits.  fp32 in, fp32
throughout: sums of up to 400 terms, so 1e-5 of a result's own size holds them with room."""
import ctypes
import importlib
import math
import os
import subprocess
import tempfile

import pytest
import torch


@pytest.fixture(scope="module")
def layers(pkg):
    return importlib.import_module(pkg.__name__ + ".layers")


def case(layers, kind, bias, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    w = layers.LmHeadWeights(weight=r(400, 64) * 0.2, gain=r(64) * 0.1, kind=kind, shift=r(64) * 0.1 if kind == "layer" else None,
                             bias=r(400) * 0.3 if bias else None, eps=1e-5)
    return g, r(3, 20, 64), w


def expected(x, w, labels, teacher, T, scale):
    """(loss, gradients) by autograd on the definition, in 64 bits."""
    leaves = {k: v.detach().double().requires_grad_() for k, v in
              dict(x=x, gain=w.gain, shift=w.shift, weight=w.weight, bias=w.bias).items() if v is not None}
    h = leaves["x"].reshape(-1, x.shape[-1])
    h = torch.nn.functional.layer_norm(h, h.shape[-1:], leaves["gain"], leaves["shift"], w.eps) if w.kind == "layer" else \
        h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + w.eps) * (1 + leaves["gain"])
    z = h @ leaves["weight"].t() + leaves.get("bias", 0.0)
    if teacher is None:
        loss = torch.nn.functional.cross_entropy(z, labels.reshape(-1), ignore_index=-100)
    else:
        index, logits = (t.reshape(-1, t.shape[-1]) for t in teacher)
        rows = (index >= 0).any(1)
        q = torch.softmax(torch.where(index >= 0, logits.double() / T, -math.inf)[rows], 1)
        logp = torch.log_softmax(z / T, 1)[rows].gather(1, index[rows].clamp(min=0))
        loss = T * T * (torch.special.xlogy(q, q) - q * logp).sum() / rows.sum()
    (loss * scale).backward()
    return loss.detach(), {k: v.grad for k, v in leaves.items()}


def targets(g, distill):
    if not distill:
        labels = torch.randint(0, 400, (3, 20), generator=g)
        labels[0, :7] = -100
        return labels, None
    index = torch.stack([torch.randperm(400, generator=g)[:9] for _ in range(60)]).view(3, 20, 9)
    index[1, :5] = -1
    index[2, :, 6:] = -1
    return None, (index, torch.randn(3, 20, 9, generator=g) * 2)


@pytest.mark.parametrize("kind,bias", [("rms", False), ("layer", True)])
@pytest.mark.parametrize("distill", [False, True])
def test_plain_pass_against_autograd(layers, kind, bias, distill):
    g, x, w = case(layers, kind, bias)
    labels, teacher = targets(g, distill)
    T = 2.0 if distill else 1.0
    loss, grads = layers.lm_head_training_pass(x, w, object(), labels=labels, teacher=teacher, temperature=T, loss_scale=3.0)
    want, wanted = expected(x, w, labels, teacher, T, 3.0)
    assert abs(loss.item() - want.item()) < 1e-5 * abs(want.item())
    for name, ref in wanted.items():
        got = getattr(grads, name).double()
        assert (got - ref).norm() <= 1e-5 * ref.norm(), name
    if not bias:
        assert grads.bias is None
    frozen = layers.lm_head_training_pass(x, w, object(), labels=labels, teacher=teacher, temperature=T, weight_grad=False)[1]
    assert frozen.weight is None and frozen.bias is None


def test_one_kind_of_target(layers):
    g, x, w = case(layers, "rms", False)
    labels, _ = targets(g, False)
    _, teacher = targets(g, True)
    for kw in ({}, {"labels": labels, "teacher": teacher}):
        with pytest.raises(ValueError):
            layers.lm_head_training_pass(x, w, object(), **kw)


def test_descriptors_are_laid_out_as_in_the_header(pkg):
    """Every field of the two descriptors: where the C compiler puts it and where ctypes does."""
    pairs = {"ixk_row_norm_desc": pkg._RowNormDesc, "ixk_linear_loss_desc": pkg._LinearLossDesc}
    lines = [f'printf("%zu\\n", sizeof({c}));' + "".join(f'printf("%zu\\n", offsetof({c}, {f[0]}));' for f in s._fields_) for c, s in pairs.items()]
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "probe.c"), os.path.join(d, "probe")
        with open(src, "w") as f:
            f.write("#include <stdio.h>\n#include <stddef.h>\n#include \"ixk.h\"\nint main(void) {" + "\n".join(lines) + "return 0; }\n")
        subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(root, "include"), src, "-o", exe], check=True)
        got = [int(v) for v in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    want = [v for s in pairs.values() for v in [ctypes.sizeof(s)] + [getattr(s, f[0]).offset for f in s._fields_]]
    assert got == want
