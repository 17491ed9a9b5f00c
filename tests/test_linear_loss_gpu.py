"""GPU: cross entropy and distillation at the vocabulary head against the definitions in 64 bits.

Bounds, derived before the first run.  u is half an ulp of the type (2^-8 bf16, 2^-11 fp16), e = 2^-24.  Logits are fp32 sums of D
exact products: within D e of S = sum |x w| (+ |b|), whatever the order; call the largest such error over a row dz, scaled
like the logits, plus 8 e of the largest logit for the base-2 exponent's rounding.  Then
  |lse - want|  <= dz + 2^-20 (1 + |lse|)              (sums of up to 2^18 terms that are each right to 2^-21)
  |loss - want| <= factor (2 dz + 2^-19 (1 + |lse| + max|z|))
  G = g (p - q): each entry within g (p (2 dz + 2^-18) + 2^-20 q) and one rounding u |G| (fp16: and 2^-24 of the largest row's g,
  the smallest step after scaling, whose own size is between 2^-14 and 2^-13 of the scaled range) =: dG
  |dx - want|  <= u |want| + sum_v dG |w| + (V + 64) e sum |G w|
  |dw - want|  <= u |want| + sum_i dG |x| + (N + 64) e sum |G x|,  db likewise
fp16 results add half of their smallest step, 2^-25."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E = 2.0 ** -24
D64 = torch.float64


def reference(x, w, b, index, q, present, scale, factor, g):
    """In 64 bits on the GPU.  index, q, present [N, K]; z = scale (x w^T + b); loss = factor * divergence."""
    x, w = x.to(D64), w.to(D64)
    active = present.any(1)
    x = torch.where(active[:, None], x, 0.0)
    bias = 0 if b is None else b.to(D64)
    z = scale * (x @ w.t() + bias)
    lse = torch.logsumexp(z, 1)
    idx = torch.where(present, index.long(), 0)
    logp = z.gather(1, idx) - lse[:, None]
    terms = torch.where(present & (q > 0), q * (torch.log(torch.where(q > 0, q, 1.0)) - logp), 0.0)
    loss = torch.where(active, factor * terms.sum(1), 0.0)
    p = torch.exp(z - lse[:, None])
    Q = torch.zeros_like(p).scatter_add_(1, idx, torch.where(present, q, 0.0))
    gg = torch.where(active, g.to(D64) * factor * scale, 0.0)[:, None]
    G = gg * (p - Q)
    # bounds
    dz = scale * (x.shape[1] * E * (x.abs() @ w.abs().t() + (0 if b is None else bias.abs()))).amax(1) + 8 * E * z.abs().amax(1)
    return dict(active=active, x=x, w=w, z=z, lse=torch.where(active, lse, 0.0), loss=loss, p=p, Q=Q, G=G, gg=gg.abs(), dz=dz, factor=factor,
                dx=G @ w, dw=G.t() @ x, db=G.sum(0))


def within(name, got, want, lim):
    err = (got.to(D64) - want).abs()
    assert got.isfinite().all(), f"{name}: not finite"
    worst = (err - lim).max().item() if err.numel() else 0.0
    assert worst <= 0, f"{name}: {worst} beyond its bound, error {err.max().item()}"


def check(r, dtype, loss, lse, grads):
    act = r["active"].to(D64)
    within("lse", lse, r["lse"], act * (r["dz"] + 2.0 ** -20 * (1 + r["lse"].abs())))
    zmax = r["z"].abs().amax(1)
    within("loss", loss, r["loss"], act * r["factor"] * (2 * r["dz"] + 2.0 ** -19 * (1 + r["lse"].abs() + zmax)) + 2.0 ** -22 * r["loss"].abs())
    if grads is None:
        return
    u, tiny = U[dtype], 2.0 ** -25 if dtype == torch.float16 else 0.0
    dG = r["gg"] * (r["p"] * (2 * r["dz"][:, None] + 2.0 ** -18) + 2.0 ** -20 * r["Q"]) + u * r["G"].abs()
    if dtype == torch.float16 and r["gg"].numel():
        dG = dG + act[:, None] * 2.0 ** -24 * 2.0 ** -13 * r["gg"].max()
    dx, dw, db = grads
    N, V = r["p"].shape
    aG, ax, aw = r["G"].abs(), r["x"].abs(), r["w"].abs()
    within("dx", dx, r["dx"], u * r["dx"].abs() + dG @ aw + (V + 64) * E * (aG @ aw) + tiny)
    if dw is not None:
        within("dw", dw, r["dw"], u * r["dw"].abs() + dG.t() @ ax + (N + 64) * E * (aG.t() @ ax) + tiny)
    if db is not None:
        within("db", db, r["db"], u * r["db"].abs() + dG.sum(0) + (N + 64) * E * aG.sum(0) + tiny)


def head(N, D, V, dtype, cuda, order="vd", bias=False, seed=0, pitch=0):
    gen = torch.Generator().manual_seed(seed + N * 7 + D * 3 + V)
    ld = (D + 7) // 8 * 8 + pitch
    x = torch.randn(N, ld, generator=gen).to(dtype).to(cuda)[:, :D]
    w = torch.randn(V, D, generator=gen) * 2.0 / math.sqrt(D)
    if order == "vd":
        store = torch.zeros(V, ld, dtype=dtype, device=cuda)
        store[:, :D] = w.to(dtype)
        w = store[:, :D]
    else:
        store = torch.zeros(D, (V + 7) // 8 * 8 + pitch, dtype=dtype, device=cuda)
        store[:, :V] = w.t().to(dtype)
        w = store[:, :V].t()
    b = (torch.randn(V, generator=gen) * 0.5).to(dtype).to(cuda) if bias else None
    g = (torch.rand(N, generator=gen) / max(N, 1) + 0.1 / max(N, 1)).to(cuda)
    return gen, x, w, b, g


# one row, one column, ends inside a slab, a tile, a group of columns, a row block; one row block and several; both kernels
XENT = [
    # N, D, V, dtype, order, bias, ignored
    (1, 8, 1, "bf16", "vd", False, 0.0),
    (1, 64, 33, "fp16", "vd", True, 0.0),
    (2, 40, 1000, "bf16", "dv", False, 0.0),
    (16, 200, 777, "bf16", "vd", True, 0.3),
    (100, 72, 513, "fp16", "dv", True, 0.5),
    (128, 128, 2000, "bf16", "vd", False, 0.0),
    (129, 64, 300, "bf16", "vd", True, 0.4),
    (200, 500, 1031, "fp16", "vd", False, 0.1),
    (257, 136, 4099, "bf16", "dv", False, 0.0),
    (700, 96, 6400, "bf16", "vd", True, 0.5),
    (1500, 64, 5003, "fp16", "vd", False, 0.3),
    (1030, 264, 20000, "bf16", "dv", True, 0.0),
    (4200, 32, 1111, "bf16", "vd", False, 0.2),
]
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def labels_for(gen, N, V, ignored, dtype=torch.int64):
    labels = torch.randint(0, V, (N,), generator=gen)
    drop = torch.rand(N, generator=gen) < ignored
    return torch.where(drop, -100, labels).to(dtype)


def one_hot_args(labels, V):
    present = ((labels >= 0) & (labels < V))[:, None]
    return labels[:, None], present.to(D64), present


@pytest.mark.parametrize("N,D,V,dtype,order,bias,ignored", XENT)
def test_cross_entropy(pkg, cuda, N, D, V, dtype, order, bias, ignored):
    gen, x, w, b, g = head(N, D, V, DT[dtype], cuda, order, bias)
    labels = labels_for(gen, N, V, ignored, torch.int32 if N % 2 else torch.int64).to(cuda)
    loss, lse = pkg.linear_cross_entropy(x, w, labels, bias=b)
    grads = pkg.linear_cross_entropy_backward(x, w, labels, lse, g, bias=b)
    assert grads[1].stride().index(1) == w.stride().index(1) or D == 1 or V == 1
    check(reference(x, w, b, *one_hot_args(labels, V), 1.0, 1.0, g), DT[dtype], loss, lse, grads)


DISTILL = [
    # N, D, V, K, dtype, order, bias, T
    (1, 8, 5, 1, "bf16", "vd", False, 1.0),
    (3, 64, 100, 7, "fp16", "vd", True, 2.0),
    (17, 104, 999, 33, "bf16", "dv", False, 4.0),
    (128, 64, 700, 256, "bf16", "vd", True, 1.5),
    (150, 72, 513, 64, "fp16", "vd", False, 2.0),
    (600, 64, 9000, 20, "bf16", "vd", False, 1.0),
    (1100, 128, 5000, 100, "bf16", "dv", True, 2.0),
]


def teacher_for(gen, N, V, K):
    index = torch.stack([torch.randperm(V, generator=gen)[:K] if V >= K else torch.randint(0, V, (K,), generator=gen) for _ in range(N)])
    return index, torch.randn(N, K, generator=gen) * 3


def teacher_args(index, logits, T, V):
    present = (index >= 0) & (index < V) & (logits > -math.inf)
    t = torch.where(present, logits.to(D64) / T, -math.inf)
    q = torch.where(present.any(1)[:, None], torch.softmax(t, 1), 0.0)
    return index, torch.where(present, q, 0.0), present


@pytest.mark.parametrize("N,D,V,K,dtype,order,bias,T", DISTILL)
def test_distillation(pkg, cuda, N, D, V, K, dtype, order, bias, T):
    gen, x, w, b, g = head(N, D, V, DT[dtype], cuda, order, bias)
    index, logits = teacher_for(gen, N, V, K)
    gone = torch.rand(N, K, generator=gen) < 0.2
    index[gone & (logits > 0)] = -1
    logits[gone & (logits <= 0)] = -math.inf
    index[:: 5] = torch.where(torch.rand(N, generator=gen)[:: 5, None] < 0.5, V + 3, index[:: 5])     # whole rows outside
    index = index.to(torch.int32 if K % 2 else torch.int64).to(cuda)
    logits = logits.to([torch.float32, DT[dtype]][N % 2]).to(cuda)
    loss, lse = pkg.linear_distillation(x, w, index, logits, bias=b, temperature=T)
    grads = pkg.linear_distillation_backward(x, w, index, logits, lse, g, bias=b, temperature=T)
    check(reference(x, w, b, *teacher_args(index, logits, T, V), 1 / T, T * T, g), DT[dtype], loss, lse, grads)


def test_entries_that_appear_twice_and_strided_entries(pkg, cuda):
    gen, x, w, b, g = head(40, 64, 300, torch.bfloat16, cuda)
    index = torch.randint(0, 20, (40, 30), generator=gen).to(cuda)[:, 5:25]
    logits = torch.randn(40, 26, generator=gen).to(cuda)[:, 3:23]
    loss, lse = pkg.linear_distillation(x, w, index, logits, temperature=2.0)
    grads = pkg.linear_distillation_backward(x, w, index, logits, lse, g, temperature=2.0)
    check(reference(x, w, b, *teacher_args(index, logits, 2.0, 300), 0.5, 4.0, g), torch.bfloat16, loss, lse, grads)


@pytest.mark.parametrize("N", [60, 300, 2000])
def test_rows_without_a_target_may_hold_anything(pkg, cuda, N):
    """NaN and infinities in the hidden states and in grad_loss of rows that do not count; labels outside the vocabulary."""
    V = 3000
    gen, x, w, b, g = head(N, 64, V, torch.bfloat16, cuda, bias=True)
    labels = labels_for(gen, N, V, 0.4).to(cuda)
    labels[3], labels[10], labels[11] = V, -1, 2 ** 40
    labels[labels == 7] = 8
    labels[20:23] = 7
    out = (labels < 0) | (labels >= V) | (labels == 7)
    clean = pkg.linear_cross_entropy(x, w, labels, bias=b, ignore_index=7)
    dirty_x = torch.where(out[:, None], torch.tensor([math.nan, math.inf], device=cuda, dtype=x.dtype).repeat(32), x)
    dirty_g = torch.where(out, math.nan, g)
    loss, lse = pkg.linear_cross_entropy(dirty_x, w, labels, bias=b, ignore_index=7)
    # (-100 is outside the vocabulary too)
    assert torch.equal(loss, clean[0]) and torch.equal(lse, clean[1]) and (loss[out] == 0).all() and (lse[out] == 0).all()
    grads = pkg.linear_cross_entropy_backward(dirty_x, w, labels, lse, dirty_g, bias=b, ignore_index=7)
    assert (grads[0][out] == 0).all()
    labels = torch.where(out, -100, labels)
    check(reference(x, w, b, *one_hot_args(labels, V), 1.0, 1.0, g), torch.bfloat16, loss, lse, grads)


@pytest.mark.parametrize("N", [5, 500])
def test_no_row_counts(pkg, cuda, N):
    gen, x, w, b, g = head(N, 64, 6000, torch.float16, cuda, bias=True)
    labels = torch.full((N,), -100, device=cuda)
    loss, lse = pkg.linear_cross_entropy(x, w, labels, bias=b)
    dx, dw, db = pkg.linear_cross_entropy_backward(x, w, labels, lse, g, bias=b)
    for t in (loss, lse, dx, dw, db):
        assert (t == 0).all()


def test_no_rows(pkg, cuda):
    gen, x, w, b, g = head(0, 64, 100, torch.bfloat16, cuda, bias=True)
    labels = torch.empty(0, dtype=torch.int64, device=cuda)
    loss, lse = pkg.linear_cross_entropy(x, w, labels, bias=b)
    dx, dw, db = pkg.linear_cross_entropy_backward(x, w, labels, lse, g, bias=b)
    assert loss.shape == (0,) and dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()


@pytest.mark.parametrize("scale", [0.25, 8.0])
def test_scaled_logits_and_confident_rows(pkg, cuda, scale):
    """At 8 the logits reach about 60 and p is 1 for single tokens: p - 1 and exponentials far below 1."""
    gen, x, w, b, g = head(300, 64, 2000, torch.bfloat16, cuda)
    labels = torch.where(torch.rand(300, generator=gen).to(cuda) < 0.5, (x.float() @ w.float().t()).argmax(1),
                         torch.randint(0, 2000, (300,), generator=gen).to(cuda))
    loss, lse = pkg.linear_cross_entropy(x, w, labels, logit_scale=scale)
    grads = pkg.linear_cross_entropy_backward(x, w, labels, lse, g, logit_scale=scale)
    check(reference(x, w, b, *one_hot_args(labels, 2000), scale, 1.0, g), torch.bfloat16, loss, lse, grads)


@pytest.mark.parametrize("big", [1.0, 2.0 ** -20, 4096.0])
def test_fp16_gradients_of_any_size(pkg, cuda, big):
    """grad_loss far below and above what fp16 holds on the way; the results' own range is the caller's."""
    gen, x, w, b, g = head(300, 64, 3000, torch.float16, cuda, bias=True)
    labels = labels_for(gen, 300, 3000, 0.1).to(cuda)
    g = g * big
    loss, lse = pkg.linear_cross_entropy(x, w, labels, bias=b)
    grads = pkg.linear_cross_entropy_backward(x, w, labels, lse, g, bias=b)
    check(reference(x, w, b, *one_hot_args(labels, 3000), 1.0, 1.0, g), torch.float16, loss, lse, grads)


def test_infinite_logits(pkg, cuda):
    """A column at -inf is a masked token; one at +inf makes its rows' lse infinite; NaN stays NaN; other rows are untouched."""
    gen, x, w, b, g = head(20, 64, 500, torch.bfloat16, cuda, bias=True)
    labels = torch.randint(100, 500, (20,), generator=gen).to(cuda)
    b[:50] = -math.inf
    loss, lse = pkg.linear_cross_entropy(x, w, labels, bias=b)
    ref = torch.logsumexp((x.double() @ w.double().t() + b.double()), 1)
    assert (lse - ref).abs().max() < 1e-4 and loss.isfinite().all()
    dx, dw, db = pkg.linear_cross_entropy_backward(x, w, labels, lse, g, bias=b)
    assert (dw[:50] == 0).all() and (db[:50] == 0).all() and dx.isfinite().all()
    b[3] = math.inf
    assert (pkg.linear_cross_entropy(x, w, labels, bias=b)[1] == math.inf).all()
    b[3] = 0
    x[4, 0] = math.nan
    again = pkg.linear_cross_entropy(x, w, labels, bias=b)[1]
    assert again[4].isnan() and again[[i for i in range(20) if i != 4]].isfinite().all()


def test_pitches_layouts_and_results_of_the_callers(pkg, cuda):
    gen, x, w, b, g = head(200, 96, 1500, torch.bfloat16, cuda, pitch=16)
    labels = labels_for(gen, 200, 1500, 0.2).to(cuda)
    loss, lse = pkg.linear_cross_entropy(x, w, labels)
    first = pkg.linear_cross_entropy_backward(x, w, labels, lse, g)
    wide = torch.full((200, 99), 5.0, dtype=x.dtype, device=cuda)
    turned = torch.full((97, 1500), 5.0, dtype=x.dtype, device=cuda)
    ws = torch.empty(pkg.linear_loss_workspace_bytes(x, w, backward=True), dtype=torch.uint8, device=cuda)
    dx, dw, db = pkg.linear_cross_entropy_backward(x, w, labels, lse, g, grad_x=wide[:, 1:97], grad_weight=turned[:96].t(), workspace=ws)
    assert torch.equal(dx, first[0]) and torch.equal(dw, first[1]) and db is None
    assert (wide[:, 0] == 5).all() and (wide[:, 97:] == 5).all() and (turned[96] == 5).all()
    frozen = pkg.linear_cross_entropy_backward(x, w, labels, lse, g, weight_grad=False)
    assert torch.equal(frozen[0], first[0]) and frozen[1] is None
    shared = pkg.linear_cross_entropy_backward(x, w, labels, lse, torch.tensor(0.25, device=cuda))
    each = pkg.linear_cross_entropy_backward(x, w, labels, lse, torch.full((200,), 0.25, device=cuda))
    assert all(torch.equal(a, c) for a, c in zip(shared[:2], each[:2]))


@pytest.mark.parametrize("N,V", [(40, 3000), (1000, 20000)])
def test_same_bits_every_time_and_on_another_stream(pkg, cuda, N, V):
    gen, x, w, b, g = head(N, 128, V, torch.bfloat16, cuda, bias=True)
    index, logits = teacher_for(gen, N, V, 16)
    index, logits = index.to(cuda), logits.to(cuda)

    def run():
        loss, lse = pkg.linear_distillation(x, w, index, logits, bias=b, temperature=2.0)
        return (loss, lse, *pkg.linear_distillation_backward(x, w, index, logits, lse, g, bias=b, temperature=2.0))

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, c, d in zip(first, run(), other):
        assert torch.equal(a, c) and torch.equal(a, d)


@pytest.mark.parametrize("distill", [False, True])
def test_gradient_against_differences(pkg, cuda, distill):
    """Central differences of the summed loss along steps that bf16 holds exactly (weights and hidden states on a grid of 1/8,
    steps of 1/4 in single entries): the loss's third derivative along an entry is at most |x|^3 < 30, so t^2 / 6 of it is
    0.3 times p (1 - p) ~ 1 / V; with V = 40 that is 8e-3 of a gradient of size up to 3, and the bf16 gradient adds 2^-7 of it."""
    gen = torch.Generator().manual_seed(9)
    N, D, V = 12, 16, 40
    x = (torch.randint(-8, 9, (N, D), generator=gen) / 8.0).bfloat16().to(cuda)
    w = (torch.randint(-8, 9, (V, D), generator=gen) / 8.0).bfloat16().to(cuda)
    labels = torch.randint(0, V, (N,), generator=gen).to(cuda)
    index, logits = (t.to(cuda) for t in teacher_for(gen, N, V, 5))
    f = (lambda a, c: pkg.linear_distillation(a, c, index, logits, temperature=2.0)) if distill else \
        (lambda a, c: pkg.linear_cross_entropy(a, c, labels))
    lse, g = f(x, w)[1], torch.ones(N, device=cuda)
    grads = pkg.linear_distillation_backward(x, w, index, logits, lse, g, temperature=2.0) if distill else \
        pkg.linear_cross_entropy_backward(x, w, labels, lse, g)
    t = 0.25
    for which, (i, j) in (("x", (3, 5)), ("x", (11, 0)), ("w", (int(labels[0]), 2)), ("w", (int(index[4, 0]), 15)), ("w", (39, 7))):
        ends = []
        for s in (t, -t):
            a, c = x.clone(), w.clone()
            (a if which == "x" else c)[i, j] += s
            ends.append(f(a, c)[0].double().sum().item())
        slope = (ends[0] - ends[1]) / (2 * t)
        grad = grads[0 if which == "x" else 1][i, j].item()
        assert abs(slope - grad) <= 0.03 + 0.01 * abs(grad), (which, i, j, slope, grad)


def test_refusals(pkg, cuda):
    gen, x, w, b, g = head(20, 64, 100, torch.bfloat16, cuda, bias=True)
    labels = torch.zeros(20, dtype=torch.int64, device=cuda)
    index, logits = torch.zeros(20, 4, dtype=torch.int64, device=cuda), torch.zeros(20, 4, device=cuda)
    loss, lse = pkg.linear_cross_entropy(x, w, labels, bias=b)
    for call in (lambda: pkg.linear_cross_entropy(x.float(), w.float(), labels), lambda: pkg.linear_cross_entropy(x, w.half(), labels),
                 lambda: pkg.linear_cross_entropy(x[:, :60], w, labels), lambda: pkg.linear_cross_entropy(x, w, labels[:19]),
                 lambda: pkg.linear_cross_entropy(x, w, labels.float()), lambda: pkg.linear_cross_entropy(x, w, labels, bias=b[:99]),
                 lambda: pkg.linear_cross_entropy(x.cpu(), w, labels), lambda: pkg.linear_cross_entropy(x, w, labels.cpu()),
                 lambda: pkg.linear_cross_entropy(x, w, labels, logit_scale=0.0), lambda: pkg.linear_cross_entropy(x, w, labels, logit_scale=math.nan),
                 lambda: pkg.linear_cross_entropy(x[:, 1:9], w[:, :8], labels),          # not 16-byte aligned
                 lambda: pkg.linear_cross_entropy(torch.zeros(20, 60, device=cuda, dtype=x.dtype), torch.zeros(100, 60, device=cuda, dtype=x.dtype), labels),
                 lambda: pkg.linear_cross_entropy(x, w, labels, workspace=torch.empty(256, dtype=torch.uint8, device=cuda)),
                 lambda: pkg.linear_distillation(x, w, index, logits[:, :3]), lambda: pkg.linear_distillation(x, w, index, logits, temperature=-1.0),
                 lambda: pkg.linear_distillation(x, w, index[:, :0], logits[:, :0]), lambda: pkg.linear_distillation(x, w, index.repeat(1, 65), logits.repeat(1, 65)),
                 lambda: pkg.linear_distillation(x, w, index, logits.double()), lambda: pkg.linear_distillation(x, w, index.t().contiguous().t(), logits),
                 lambda: pkg.linear_cross_entropy_backward(x, w, labels, lse[:5], g), lambda: pkg.linear_cross_entropy_backward(x, w, labels, lse, g.double()),
                 lambda: pkg.linear_cross_entropy_backward(x, w, labels, lse, g, grad_x=x[:, :8]),
                 lambda: pkg.linear_cross_entropy_backward(x, w, labels, lse, g, grad_weight=w[:50]),
                 lambda: pkg.linear_cross_entropy_backward(x, w, labels, lse, g, workspace=torch.empty(1024, dtype=torch.uint8, device=cuda))):
        with pytest.raises(pkg.IxkError):
            call()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("N", [100, 300])
def test_a_mean_leaves_the_labels_entry_whole(pkg, cuda, dtype, N):
    """With equal grad_loss a label's entry is p - 1 before its rounding, whose error is then at most p where p is small: 1 / N is
    not rounded with it."""
    V = 4096
    gen, x, w, b, g = head(N, 64, V, DT[dtype], cuda)
    x = x * 0.0625      # (p about 1 / 4096)
    labels = torch.randint(0, V, (N,), generator=gen).to(cuda)
    g = torch.full((N,), 1.0 / N, device=cuda)
    loss, lse = pkg.linear_cross_entropy(x, w, labels)
    dx, dw = pkg.linear_cross_entropy_backward(x, w, labels, lse, g)[:2]
    r = reference(x, w, None, *one_hot_args(labels, V), 1.0, 1.0, g)
    u = U[DT[dtype]]
    dG = r["gg"] * (r["p"] * (2 * r["dz"][:, None] + 2.0 ** -18) + 2.0 ** -20 * r["Q"]) + u * r["gg"] * r["p"] + 2.0 ** -37 * r["gg"]
    assert r["p"].max() < 2.0 ** -10
    tiny = 2.0 ** -25 if dtype == "fp16" else 0.0
    within("dx", dx, r["dx"], u * r["dx"].abs() + dG @ r["w"].abs() + (V + 64) * E * (r["G"].abs() @ r["w"].abs()) + tiny + r["gg"] * (r["p"] * r["Q"]).sum(1, keepdim=True) * r["w"].abs()[labels])
    within("dw", dw, r["dw"], u * r["dw"].abs() + (dG + r["gg"] * r["p"] * r["Q"]).t() @ r["x"].abs() + (N + 64) * E * (r["G"].abs().t() @ r["x"].abs()) + tiny)
