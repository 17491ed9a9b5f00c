"""CPU: the plain torch forms of the layers' glue."""
import importlib

import pytest
import torch


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_half_split_rotation_of_any_type(pkg, dtype):
    """Both halves of a pair turn by the angle that they had before either was stored.  Two roundings of a result of at most the
    pair's size (fp32 products and sum, then the store)."""
    layers = importlib.import_module(pkg.__name__ + ".layers")
    x = torch.randn(3, 2, 24, generator=torch.Generator().manual_seed(0)).to(dtype)
    cos, sin = layers.rotary_tables(torch.tensor([0, 5, 90]), 16)
    a, b, rest = x.double().split((8, 8, 8), -1)
    c, s = cos.double()[:, None], sin.double()[:, None]
    want = torch.cat((a * c - b * s, b * c + a * s, rest), -1)
    got = layers.apply_rotary_half_(x.clone(), cos, sin, 16).double()
    size = torch.cat((a.abs() + b.abs(), a.abs() + b.abs(), rest.abs()), -1)
    assert bool(((got - want).abs() <= size * (torch.finfo(dtype).eps / 2 + 3 * 2 ** -24)).all())
