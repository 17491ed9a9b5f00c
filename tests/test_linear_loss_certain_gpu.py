"""GPU: tokens that the model is sure of, at a hidden size of 4096, against the definitions in 64 bits.

With 1 - p of 1e-2 to 1e-4 the entry p - 1 of dloss/dlogits is a small difference, and what the logit of 15 that it is made of has
lost shows in it.  Bounds, derived before the first run.  e = 2^-24, u half an ulp of the type (2^-8 bf16, 2^-11 fp16).  An fp32 sum
of 4096 products, 150 additions one after the other at most with partial sums below 16, is off by sqrt(150) 16 e = 1.2e-5 (the
roundings are independent and of either sign), and an lse of 16 is held to 16 e; 2^-16 holds both.  So, per unit of grad_loss,
  |G - want| <= 2^-16 at targets, 2^-13 p elsewhere (logits off by 6e-5, and 2^-21 of the exponential), and one rounding u |G|
  |dx - want| <= u |want| + sum_v dG |w| + 2^-20 sum |G w|, db likewise with the sum over the rows
and the loss, factor * (lse - logit), is within 2^-16 of itself, and of no sign that it cannot have beyond that.  fp16 adds its smallest steps as in
test_linear_loss_gpu.py."""
import pytest
import torch

from test_linear_loss_gpu import DT, U, one_hot_args, reference, teacher_args, within

pytestmark = pytest.mark.gpu
D, V = 4096, 1504
D64 = torch.float64


def certain(N, dtype, order, cuda, seed=0):
    """Rows whose labels (distinct columns up to V) stand so far above the others that 1 - p goes from 1e-2 to 1e-4."""
    gen = torch.Generator().manual_seed(seed + N)
    w = (torch.randn(V, D, generator=gen) * 0.02).to(dtype).to(cuda)
    labels = torch.randperm(V, generator=gen)[:N].to(cuda)
    x = (torch.randn(N, D, generator=gen) * 0.5).to(cuda)
    want = 10.0 ** -(2.0 + 2.0 * torch.rand(N, generator=gen)).to(cuda).to(D64)
    w64 = w.to(D64)
    for _ in range(2):      # (twice: the second time the rest of the row is known)
        z = x.to(D64) @ w64.t()
        own = z.gather(1, labels[:, None])
        rest = torch.logsumexp(z.scatter(1, labels[:, None], -torch.inf), 1, keepdim=True)
        lift = rest + torch.log(1 / want[:, None] - 1) - own
        x = x + (lift / (w64[labels] ** 2).sum(1, keepdim=True)).float() * w[labels].float()
    w = w if order == "vd" else w.t().contiguous().t()
    return gen, x.to(dtype), w, labels


def check(r, dtype, loss, grads, loss_size):
    u, gg = U[dtype], r["gg"]
    dG = gg * torch.where(r["Q"] > 0, 2.0 ** -16, 2.0 ** -13 * r["p"]) + u * r["G"].abs()
    tiny = 0.0
    if dtype == torch.float16:
        dG, tiny = dG + 2.0 ** -37 * gg.max(), 2.0 ** -25
    within("loss", loss, r["loss"], r["factor"] * loss_size * 2.0 ** -16)
    dx, _, db = grads
    aG, aw = r["G"].abs(), r["w"].abs()
    within("dx", dx, r["dx"], u * r["dx"].abs() + dG @ aw + 2.0 ** -20 * (aG @ aw) + tiny)
    within("db", db, r["db"], u * r["db"].abs() + dG.sum(0) + 2.0 ** -20 * aG.sum(0) + tiny)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("order", ["vd", "dv"])
@pytest.mark.parametrize("N", [50, 200, 1100])
def test_cross_entropy(pkg, cuda, dtype, order, N):
    gen, x, w, labels = certain(N, DT[dtype], order, cuda)
    b = torch.zeros(V, dtype=x.dtype, device=cuda)
    g = torch.full((N,), 1.0, device=cuda)
    loss, lse = pkg.linear_cross_entropy(x, w, labels, bias=b)
    grads = pkg.linear_cross_entropy_backward(x, w, labels, lse, g, bias=b)
    r = reference(x, w, b, *one_hot_args(labels, V), 1.0, 1.0, g)
    rest = 1 - r["p"].gather(1, labels[:, None])
    assert rest.max() < 2e-2 and rest.min() < 1e-3 and rest.min() > 1e-5
    check(r, x.dtype, loss, grads, 1.0)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("N", [50, 200])
def test_distillation_from_a_teacher_that_agrees(pkg, cuda, dtype, N):
    """The teacher's entries are the student's four largest logits, give or take 1e-3: p and q differ by as little."""
    gen, x, w, labels = certain(N, DT[dtype], "vd", cuda, seed=1)
    b = torch.zeros(V, dtype=x.dtype, device=cuda)
    g = torch.full((N,), 1.0, device=cuda)
    top = (x.to(D64) @ w.to(D64).t()).topk(4, 1)
    index, logits = top.indices, (top.values + 1e-3 * torch.randn(N, 4, generator=gen).to(cuda)).float()
    loss, lse = pkg.linear_distillation(x, w, index, logits, bias=b)
    grads = pkg.linear_distillation_backward(x, w, index, logits, lse, g, bias=b)
    r = reference(x, w, b, *teacher_args(index, logits, 1.0, V), 1.0, 1.0, g)
    check(r, x.dtype, loss, grads, 1.0)


@pytest.mark.parametrize("order", ["vd", "dv"])
@pytest.mark.parametrize("N", [60, 300, 700, 4200])
def test_losses_next_to_zero(pkg, cuda, order, N):
    """1 - p from 1e-3 down to 1e-9: no loss is below 0, and where the label's logit is a product of its own (row-major, or up to
    128 rows) a loss is right to 2^-12 of itself: its terms' logits are off by up to 6e-5 each way, their exponentials by 2^-21."""
    gen = torch.Generator().manual_seed(N)
    d, v = 1024, 1000
    w = (torch.randn(v, d, generator=gen) * 0.04).bfloat16().to(cuda)
    labels = torch.randint(0, v, (N,), generator=gen).to(cuda)
    lift = (15.0 + 15.0 * torch.rand(N, 1, generator=gen)).to(cuda) / (0.0016 * d)
    x = ((torch.randn(N, d, generator=gen) * 0.5).to(cuda) + lift * w[labels].float()).bfloat16()
    z = x.to(D64) @ w.to(D64).t()
    rest = torch.logsumexp(z.scatter(1, labels[:, None], -torch.inf), 1) - z.gather(1, labels[:, None])[:, 0]
    want = torch.log1p(torch.exp(rest))
    assert want.min() < 1e-7 and want.max() > 1e-4
    loss, lse = pkg.linear_cross_entropy(x, w if order == "vd" else w.t().contiguous().t(), labels)
    assert (loss >= 0).all()
    assert (lse.to(D64) - torch.logsumexp(z, 1)).abs().max() < 2.0 ** -13
    if order == "vd" or N <= 128:
        assert ((loss.to(D64) - want).abs() <= 2.0 ** -12 * want).all()
