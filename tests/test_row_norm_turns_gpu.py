"""GPU: row norms of sizes at which a CTA has more than one turn: the ring's stages filled again, two rows a batch, sums over
several rows a CTA of the columns above 8192, several rounds of short rows.  The bounds of test_row_norm_training_gpu.py."""
import pytest
import torch

from test_row_norm_training_gpu import check

pytestmark = pytest.mark.gpu

SIZES = [(5000, 1000), (3000, 4096), (3000, 2047), (700, 8200), (700, 12287), (60000, 64), (9000, 300), (20000, 33), (2500, 8192), (40001, 256)]


@pytest.mark.parametrize("dtype,param", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_against_64_bits(pkg, cuda, dtype, param, kind, rows, cols):
    gen = torch.Generator(device=cuda).manual_seed(rows * 1000 + cols)
    r = lambda *s: torch.randn(*s, generator=gen, device=cuda)  # noqa: E731
    x, g, off = (r(rows, cols) * 1.5 + 0.4).to(dtype), r(rows, cols).to(dtype), float(kind)
    gain, shift = (r(cols) * 0.2 + 1 - off).to(param), (r(cols) * 0.2).to(param)
    y, mean, rstd = pkg.row_norm_forward(x, kind=kind, eps=1e-5, gain=gain, gain_offset=off, shift=shift)
    dx, dgain, dshift = pkg.row_norm_backward(g, x, mean, rstd, kind=kind, gain=gain, gain_offset=off, with_shift=True)
    check(pkg, x, g, kind, gain, off, shift, 1e-5, y, mean, rstd, dx, dgain, dshift)
    # and in place, with the same bits
    again = g.clone()
    assert torch.equal(pkg.row_norm_backward(again, x, mean, rstd, kind=kind, gain=gain, gain_offset=off, grad_x=again)[0], dx)
    over = x.clone()
    assert torch.equal(pkg.row_norm_forward(over, kind=kind, eps=1e-5, gain=gain, gain_offset=off, shift=shift, out=over)[0], y)


@pytest.mark.parametrize("cols,at", [(2040, 1), (2047, 3), (9000, 2), (300, 5)])
def test_rows_apart_at_odd_addresses(pkg, cuda, cols, at):
    """Rows that start anywhere within 16 bytes, several turns; what lies between them stays as it was."""
    gen = torch.Generator(device=cuda).manual_seed(cols)
    rows, pitch = 3001, cols + 11
    r = lambda *s: torch.randn(*s, generator=gen, device=cuda)  # noqa: E731
    wide_x, wide_g, out = r(rows, pitch).bfloat16(), r(rows, pitch).bfloat16(), torch.full((rows, pitch), 7.0, device=cuda, dtype=torch.bfloat16)
    x, g, gain = wide_x[:, at:at + cols], wide_g[:, at:at + cols], (r(cols) * 0.2 + 1).bfloat16()
    y, mean, rstd = pkg.row_norm_forward(x, eps=1e-5, gain=gain)
    dx, dgain, dshift = pkg.row_norm_backward(g, x, mean, rstd, gain=gain, with_shift=True, grad_x=out[:, at:at + cols])
    assert (out[:, :at] == 7).all() and (out[:, at + cols:] == 7).all()
    check(pkg, x, g, 0, gain, 0.0, None, 1e-5, y, mean, rstd, dx, dgain, dshift)
