"""quantize_rows' codes, on the CPU."""

import math

import torch

from conftest import load_package

dn = load_package()


def test_codes_of_the_smallest_values_are_finite():
    """A row whose scale is the smallest number of fp32, and stands for 1.4 of it."""
    tiny = 2.0 ** -149
    t = (torch.arange(-627, 628, dtype=torch.float64) * tiny).float()[None]
    q = dn.quantize_rows(t)
    assert q.scale.double().item() == tiny
    codes = q.codes.float()
    assert torch.isfinite(codes).all() and codes.abs().max() == 448
    assert torch.equal(codes[0, 627 - 16:627 + 17], torch.arange(-16.0, 17.0))


def test_codes_of_ordinary_empty_and_non_finite_rows():
    g = torch.Generator().manual_seed(1)
    t = torch.randn(5, 40, generator=g)
    t[1] = 0
    t[2, 3], t[3, 4] = math.nan, math.inf
    q = dn.quantize_rows(t)
    assert q.codes.stride(0) == 48 and not q.codes[1].float().any() and q.scale[1] == 0
    back = q.codes.float() * q.scale[:, None]
    for i in (0, 4):  # half a step of e4m3: 2^-4 of a normal code, 2^-10 below 2^-6
        step = torch.maximum(t[i].abs() / 16, q.scale[i] * 2.0 ** -10)
        assert ((back[i] - t[i]).abs() <= 1.01 * step).all() and q.codes[i].float().abs().max() == 448
    assert torch.isnan(back[2, 3]) and torch.isnan(back[3, 4])
