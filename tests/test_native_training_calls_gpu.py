"""GPU: the native calls of the training operators and the Python code behind them: the same bits and number of launches for
what they take, the same errors for what they refuse."""
import pytest
import torch

from test_native_calls_gpu import both, rnd

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def norm_calls(pkg):
    x, gain, shift = rnd(5, 7, 512), rnd(512), rnd(512, seed=1)
    wide = rnd(40, 100)[:, :96]

    def back(x, kind=0, gain=None, with_shift=False, fwd=None, grad=None, **kw):
        y, mean, rstd = fwd or pkg.row_norm_forward(x, kind=kind, gain=gain)
        g = rnd(*x.shape, dtype=x.dtype, seed=3) if grad is None else grad
        return [t for t in pkg.row_norm_backward(g, x, mean, rstd, kind=kind, gain=gain, with_shift=with_shift, **kw) if t is not None]

    yield "forward", lambda: [*pkg.row_norm_forward(x, gain=gain, shift=shift), *pkg.row_norm_forward(wide)]
    yield "rms", lambda: [t for t in pkg.row_norm_forward(x.half(), kind=1, eps=1e-6, gain=gain.float(), gain_offset=1) if t is not None]
    yield "into", lambda: list(pkg.row_norm_forward(wide, out=torch.empty(40, 99, dtype=BF16, device="cuda")[:, :96], stream=torch.cuda.current_stream()))
    yield "backward", lambda: back(x) + back(x, gain=gain, with_shift=True) + back(wide, 1, gain[:96].float())
    yield "backward with scratch", lambda: back(x, gain=gain, workspace=torch.empty(1 << 20, dtype=torch.uint8, device="cuda"),
                                                grad_x=torch.empty_like(x), stream=torch.cuda.current_stream())
    yield "backward on a stream", lambda: back(x, gain=gain, with_shift=True, stream=torch.cuda.current_stream())
    yield "no rows", lambda: list(pkg.row_norm_forward(x[:0], gain=gain)) + back(x[:0], gain=gain)
    fwd = pkg.row_norm_forward(x)
    for name, bad in (("layout", lambda: pkg.row_norm_forward(x.transpose(0, 1))), ("type", lambda: pkg.row_norm_forward(x.double())),
                      ("kind", lambda: pkg.row_norm_forward(x, kind=2)), ("gain", lambda: pkg.row_norm_forward(x, gain=gain[:8])),
                      ("gain type", lambda: pkg.row_norm_forward(x, gain=gain.half())), ("shift type", lambda: pkg.row_norm_forward(x, gain=gain, shift=shift.float())),
                      ("out", lambda: pkg.row_norm_forward(x, out=x[0])), ("host", lambda: pkg.row_norm_forward(x.cpu())), ("eps", lambda: pkg.row_norm_forward(x, eps=-1.0)),
                      ("length", lambda: pkg.row_norm_forward(torch.empty(1, 20000, device="cuda"))), ("grad", lambda: back(x, grad=x.float())),
                      ("mean", lambda: back(x, fwd=(x, None, fwd[2]))), ("rstd", lambda: back(x, fwd=(x, fwd[1], fwd[2][:2]))),
                      ("grad_x", lambda: back(x, grad_x=x[0])), ("scratch", lambda: back(x, gain=gain, workspace=torch.empty(16, dtype=torch.uint8, device="cuda")))):
        yield f"refused: {name}", lambda bad=bad: list(bad())


def loss_calls(pkg):
    x, w, b = rnd(50, 64), rnd(300, 64), rnd(300)
    turned = rnd(64, 304).t()[:300]
    labels = torch.arange(50, device="cuda") * 5
    index, teacher = labels[:, None] + torch.arange(4, device="cuda"), rnd(50, 4, dtype=F32)
    g = rnd(50, dtype=F32).abs()
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    some = lambda ts: [t for t in ts if t is not None]  # noqa: E731

    def xent(x=x, w=w, labels=labels, g=g, bias=None, scale=1.0, lse=None, **kw):
        loss, made = pkg.linear_cross_entropy(x, w, labels, bias=bias, logit_scale=scale)
        return [loss, made, *some(pkg.linear_cross_entropy_backward(x, w, labels, made if lse is None else lse, g, bias=bias, logit_scale=scale, **kw))]

    def distill(index=index, teacher=teacher, T=2.0, **kw):
        loss, lse = pkg.linear_distillation(x, w, index, teacher, temperature=T)
        return [loss, lse, *some(pkg.linear_distillation_backward(x, w, index, teacher, lse, g, temperature=T, **kw))]

    yield "cross entropy", lambda: xent() + xent(bias=b, scale=2) + xent(w=turned) + xent(labels=labels.int())
    yield "into", lambda: xent(grad_x=torch.empty(50, 70, dtype=BF16, device="cuda")[:, :64], grad_weight=torch.empty(64, 300, dtype=BF16, device="cuda").t(), workspace=ws)
    yield "frozen", lambda: xent(bias=b, weight_grad=False)
    yield "one for all", lambda: xent(g=torch.tensor(0.5, device="cuda")) + xent(g=torch.tensor([0.5], device="cuda").expand(50))
    yield "stream", lambda: xent(stream=torch.cuda.current_stream()) + xent(stream=torch.cuda.current_stream(), workspace=ws)
    yield "fp16", lambda: xent(x=x.half(), w=w.half())
    yield "distillation", lambda: distill() + distill(teacher=teacher.half()) + distill(index=index.int(), T=1) + distill(teacher=rnd(50, 9, dtype=F32)[:, 2:6])
    yield "no rows", lambda: xent(x=x[:0], labels=labels[:0], g=g[:0])
    for name, bad in (("shape", lambda: xent(x=x[:, :32])), ("type", lambda: xent(x=x.float(), w=w.float())), ("types", lambda: xent(w=w.half())), ("rank", lambda: xent(w=w[0])),
                      ("labels", lambda: xent(labels=labels[:3])), ("label type", lambda: xent(labels=labels.float())), ("bias", lambda: xent(bias=b[:7])),
                      ("host", lambda: xent(labels=labels.cpu())), ("scale", lambda: xent(scale=0.0)), ("lse", lambda: xent(lse=g[:9])), ("g", lambda: xent(g=g[:9])),
                      ("g type", lambda: xent(g=g.double())), ("grad_x", lambda: xent(grad_x=x[:9])), ("grad_weight", lambda: xent(grad_weight=w[:9])),
                      ("scratch", lambda: xent(workspace=ws[:512])), ("entries", lambda: distill(index=index[:, :3])), ("teacher", lambda: distill(teacher=teacher.double())),
                      ("temperature", lambda: distill(T=-2.0)), ("many", lambda: distill(index=index.repeat(1, 70), teacher=teacher.repeat(1, 70)))):
        yield f"refused: {name}", bad


@pytest.mark.parametrize("family", [norm_calls, loss_calls])
def test_native_calls_and_their_python_twins(pkg, cuda, monkeypatch, family):
    for name, call in family(pkg):
        (a, la), (b, lb) = both(pkg, monkeypatch, call)
        assert la == lb, name
        if isinstance(a, tuple) or isinstance(b, tuple):
            assert a == b and name.startswith("refused"), (name, a, b)
        else:
            assert not name.startswith("refused"), name
            assert all(torch.equal(s, t) for s, t in zip(a, b)) and len(a) == len(b) and a, name
