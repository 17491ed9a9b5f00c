"""GPU: row norms for training (row_norm_forward, row_norm_backward) against the formulas in 64 bits.

Bounds, derived before the first run.  u is the type's rounding (half an ulp, relative: 2^-8 bf16, 2^-11 fp16, 2^-24 fp32),
e = 2^-24 that of the fp32 arithmetic.  A row's sums take at most 16 terms in sequence and 10 levels of a tree, its rsqrt two
ulps: statistics are within 64 e of their size, so
  |y - want|  <= u |want| + 64 e (max|x| rstd |scale| + |shift|)
  |dx - want| <= u |want| + 128 e rstd max|h| (1 + max|xh|)^2
and a sum over R rows, whatever its order, within (R + 64) e of the sum of the terms' sizes (with the terms' own
64 e (1 + max|x| rstd) in it).  fp16 adds half of its smallest step, 2^-25."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
E = 2.0 ** -24
D64 = torch.float64

# a warp's rows and a CTA's, whole vectors and single elements, every number of elements per thread, one column, one row
SIZES = [(1, 1), (1, 8), (3, 7), (5, 64), (37, 200), (300, 256), (9, 33), (2, 255), (4, 257), (65, 264), (129, 520), (7, 1023), (64, 4096),
         (33, 2047), (3, 8192), (2, 8200), (2, 9001), (3, 16384), (1000, 48)]


def bound(got, want, slack):
    u, tiny = U[got.dtype], TINY[got.dtype]
    err = (got.double() - want).abs()
    lim = u * want.abs() * (1 + 2.0 ** -20) + slack + tiny
    worst = (err - lim).max().item()
    assert worst <= 0, f"{worst} beyond the bound, error {err.max().item()}"


def reference(x, g, kind, gain, off, shift, eps):
    x, g = x.double(), g.double()
    c = x.shape[1]
    scale = torch.ones(c, dtype=D64, device=x.device) if gain is None else gain.double() + off
    mean = x.sum(1, keepdim=True) / c if kind == 0 else torch.zeros_like(x[:, :1])
    rstd = 1 / torch.sqrt(((x - mean) ** 2).sum(1, keepdim=True) / c + eps)
    xh = (x - mean) * rstd
    y = xh * scale + (0 if shift is None else shift.double())
    h = g * scale
    dx = rstd * (h - (h.mean(1, keepdim=True) if kind == 0 else 0) - xh * (h * xh).mean(1, keepdim=True))
    return {"scale": scale, "mean": mean, "rstd": rstd, "xh": xh, "y": y, "h": h, "dx": dx, "dgain": (g * xh).sum(0), "dshift": g.sum(0)}


def check(pkg, x, g, kind, gain, off, shift, eps, y, mean, rstd, dx, dgain, dshift):
    r = reference(x, g, kind, gain, off, shift, eps)
    R = x.shape[0]
    size = x.double().abs().amax(1, keepdim=True) * r["rstd"]
    bound(rstd, r["rstd"][:, 0], 64 * E * r["rstd"][:, 0] * (1 + size[:, 0] ** 2))
    if kind == 0:
        bound(mean, r["mean"][:, 0], 64 * E * x.double().abs().amax(1))
    sh = 0 if shift is None else shift.double().abs()
    # (rstd's own error where the mean is far above the spread)
    bound(y, r["y"], 64 * E * (size * r["scale"].abs() * (1 + size) + sh))
    hm = r["h"].abs().amax(1, keepdim=True)
    bound(dx, r["dx"], 128 * E * r["rstd"] * hm * (1 + size) ** 2)
    if gain is not None:
        terms = (g.double().abs() * (r["xh"].abs() + 64 * (1 + size) ** 2 / (R + 64))).sum(0)
        bound(dgain, r["dgain"], (R + 64) * E * terms)
    if dshift is not None:
        bound(dshift, r["dshift"], (R + 64) * E * g.double().abs().sum(0))


@pytest.mark.parametrize("dtype,param", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_against_64_bits(pkg, cuda, dtype, param, kind, rows, cols):
    gen = torch.Generator().manual_seed(rows * 1000 + cols)
    x = (torch.randn(rows, cols, generator=gen) * 1.5 + 0.4).to(dtype).to(cuda)
    g = torch.randn(rows, cols, generator=gen).to(dtype).to(cuda)
    off = float(kind)
    gain = (torch.randn(cols, generator=gen) * 0.2 + 1 - off).to(param).to(cuda)
    shift = (torch.randn(cols, generator=gen) * 0.2).to(param).to(cuda)
    y, mean, rstd = pkg.row_norm_forward(x, kind=kind, eps=1e-5, gain=gain, gain_offset=off, shift=shift)
    assert (mean is None) == (kind == 1) and y.dtype == dtype and rstd.shape == (rows,)
    dx, dgain, dshift = pkg.row_norm_backward(g, x, mean, rstd, kind=kind, gain=gain, gain_offset=off, with_shift=True)
    assert dgain.dtype == param and dshift.dtype == param
    check(pkg, x, g, kind, gain, off, shift, 1e-5, y, mean, rstd, dx, dgain, dshift)


@pytest.mark.parametrize("kind", [0, 1])
def test_without_parameters(pkg, cuda, kind):
    gen = torch.Generator().manual_seed(5)
    x, g = (torch.randn(6, 40, 96, generator=gen).bfloat16().to(cuda) for _ in range(2))
    y, mean, rstd = pkg.row_norm_forward(x, kind=kind, eps=1e-6)
    dx, dgain, dshift = pkg.row_norm_backward(g, x, mean, rstd, kind=kind)
    assert dgain is None and dshift is None and rstd.shape == (6, 40)
    f = lambda t: None if t is None else t.reshape(240, *t.shape[2:])  # noqa: E731
    check(pkg, f(x), f(g), kind, None, 0.0, None, 1e-6, f(y), f(mean), f(rstd), f(dx), None, None)


@pytest.mark.parametrize("cols,pad", [(96, 8), (96, 3), (640, 24), (511, 1)])
def test_row_pitches_and_in_place(pkg, cuda, cols, pad):
    """Rows apart in memory, at addresses that no vector load takes; the memory between them stays as it was."""
    gen = torch.Generator().manual_seed(cols + pad)
    wide = torch.randn(50, cols + pad, generator=gen).half().to(cuda)
    x = wide[:, pad // 2:pad // 2 + cols]
    g = torch.randn(50, cols, generator=gen).half().to(cuda)
    gain = torch.randn(cols, generator=gen).half().to(cuda)
    out = torch.full((50, cols + pad), 7.0, dtype=torch.float16, device=cuda)
    y, mean, rstd = pkg.row_norm_forward(x, gain=gain, out=out[:, :cols])
    assert (out[:, cols:] == 7).all()
    dx, dgain, dshift = pkg.row_norm_backward(g, x, mean, rstd, gain=gain, with_shift=True)
    check(pkg, x, g, 0, gain, 0.0, None, 1e-5, y, mean, rstd, dx, dgain, dshift)
    again = g.clone()
    pkg.row_norm_backward(again, x, mean, rstd, gain=gain, grad_x=again)
    assert torch.equal(again, dx)
    before = x.clone()      # (at another address than x: sums in another order, so compared with its like)
    apart = pkg.row_norm_forward(before, gain=gain)[0]
    assert torch.equal(pkg.row_norm_forward(before, gain=gain, out=before)[0], apart)


@pytest.mark.parametrize("rows,cols", [(4000, 256), (2000, 1000), (1, 64)])
def test_same_bits_every_time_and_on_another_stream(pkg, cuda, rows, cols):
    gen = torch.Generator().manual_seed(rows)
    x, g = (torch.randn(rows, cols, generator=gen).bfloat16().to(cuda) for _ in range(2))
    gain = torch.randn(cols, generator=gen).to(cuda)
    run = lambda **kw: pkg.row_norm_backward(g, x, *pkg.row_norm_forward(x, gain=gain, **kw)[1:], gain=gain, with_shift=True, **kw)  # noqa: E731
    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(first, run(), other):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_no_rows(pkg, cuda):
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=cuda)
    gain = torch.ones(64, device=cuda)
    y, mean, rstd = pkg.row_norm_forward(x, gain=gain)
    dx, dgain, dshift = pkg.row_norm_backward(x, x, mean, rstd, gain=gain, with_shift=True)
    assert y.shape == dx.shape == (0, 64) and (dgain == 0).all() and (dshift == 0).all()


@pytest.mark.parametrize("kind", [0, 1])
def test_far_mean_and_outliers(pkg, cuda, kind):
    """A mean a thousand times the spread, and one channel a thousand times the others: no cancellation in the variance."""
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(20, 300, generator=gen).to(cuda)
    x[:10] += 1000.0
    x[10:, 0] = 1000.0
    g = torch.randn(20, 300, generator=gen).to(cuda)
    y, mean, rstd = pkg.row_norm_forward(x, kind=kind)
    dx, _, _ = pkg.row_norm_backward(g, x, mean, rstd, kind=kind)
    check(pkg, x, g, kind, None, 0.0, None, 1e-5, y, mean, rstd, dx, None, None)


def test_bad_values_stay_in_their_row(pkg, cuda):
    x = torch.randn(9, 128, device=cuda).bfloat16()
    clean = pkg.row_norm_forward(x)[0]
    x[2, 5], x[4, 7] = float("nan"), float("inf")
    y, mean, rstd = pkg.row_norm_forward(x)
    dx = pkg.row_norm_backward(x.nan_to_num(0, 0, 0), x, mean, rstd)[0]
    rest = [0, 1, 3, 5, 6, 7, 8]
    assert torch.equal(y[rest], clean[rest]) and dx[rest].isfinite().all()
    assert y[2].isnan().all() and dx[2].isnan().all()


@pytest.mark.parametrize("kind", [0, 1])
def test_gradient_against_differences(pkg, cuda, kind):
    """d/dt of sum(w . y(x + t d)) by central differences of the fp32 forward: t = 1e-2 leaves t^2 / 6 of the third
    derivative (about 1e-4 of the value here) and 2^-24 / t of the forward's rounding; 2e-3 of the gradient's size holds both."""
    gen = torch.Generator().manual_seed(11)
    x, w, d = (torch.randn(4, 96, generator=gen, dtype=D64).float().to(cuda) for _ in range(3))
    gain, shift = (torch.randn(96, generator=gen).to(cuda) for _ in range(2))
    dgain_dir = torch.randn(96, generator=gen).to(cuda)
    f = lambda xx, gg, ss: (pkg.row_norm_forward(xx, kind=kind, gain=gg, shift=ss)[0].double() * w.double()).sum().item()  # noqa: E731
    _, mean, rstd = pkg.row_norm_forward(x, kind=kind, gain=gain, shift=shift)
    dx, dgain, dshift = pkg.row_norm_backward(w, x, mean, rstd, kind=kind, gain=gain, with_shift=True)
    t = 1e-2
    for grad, direction, at in ((dx, d, lambda s: (x + s * d, gain, shift)), (dgain, dgain_dir, lambda s: (x, gain + s * dgain_dir, shift)),
                                (dshift, dgain_dir, lambda s: (x, gain, shift + s * dgain_dir))):
        slope = (f(*at(t)) - f(*at(-t))) / (2 * t)
        size = (grad.double().norm() * direction.double().norm()).item()
        assert abs(slope - (grad.double() * direction.double()).sum().item()) <= 2e-3 * size


def test_refusals(pkg, cuda):
    x = torch.randn(4, 64, device=cuda).bfloat16()
    y, mean, rstd = pkg.row_norm_forward(x)
    E_ = pkg.IxkError
    for call in (lambda: pkg.row_norm_forward(x.double()), lambda: pkg.row_norm_forward(x.cpu()), lambda: pkg.row_norm_forward(x.t()),
                 lambda: pkg.row_norm_forward(x, kind=7), lambda: pkg.row_norm_forward(x, gain=torch.ones(63, device=cuda)),
                 lambda: pkg.row_norm_forward(x, gain=torch.ones(64, device=cuda, dtype=torch.float16)),
                 lambda: pkg.row_norm_forward(x, out=torch.empty(4, 63, device=cuda, dtype=x.dtype)),
                 lambda: pkg.row_norm_forward(torch.empty(2, 16392, device=cuda)), lambda: pkg.row_norm_forward(x, eps=-1.0),
                 lambda: pkg.row_norm_backward(x[:3], x, mean, rstd), lambda: pkg.row_norm_backward(x.float(), x, mean, rstd),
                 lambda: pkg.row_norm_backward(x, x, None, rstd), lambda: pkg.row_norm_backward(x, x, mean, rstd.half()),
                 lambda: pkg.row_norm_backward(x, x, mean, rstd, with_shift=True, workspace=torch.empty(16, dtype=torch.uint8, device=cuda))):
        with pytest.raises(E_):
            call()
