"""GELU that keeps its input in 8 bits: the negative branch against 64 bits, relative to itself (there an absolute bound of 1e-7 says
nothing: from -5.5 on a result of zero would meet it)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24
# how far the fit of Phi(-a) may be off, of itself, down to -a
PHI = [(2.0, 7e-7), (4.0, 6e-6), (6.0, 4e-5), (8.0, 3.2e-4), (10.0, 1.2e-3), (12.9, 1e-2)]


@pytest.fixture(scope="module")
def c8(native):
    from beatsaberrl_b200 import checkpoint8
    return checkpoint8


def tail(t):
    """Phi(-t) in 64 bits, as exact in the tail as near zero (ndtr is not)."""
    return 0.5 * torch.erfc(t / math.sqrt(2))


def fit_error(a):
    e = torch.full_like(a, math.nan)
    for most, part in reversed(PHI):
        e = torch.where(a <= most, part, e)
    return e


def rounding(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tail_of_the_values(c8, dtype):
    """One value per row from -0.01 to -12.9: |x| Phi(-|x|), the fit's error and two roundings (the exponential's argument is part of the fit's
    figure), then the type's."""
    x = -torch.linspace(0.01, 12.9, 400001, device="cuda").to(dtype)
    x = x[x >= -12.9].view(-1, 1)
    y, _ = c8.gelu8_forward(x)
    a = -x.double()
    want = -a * tail(a)
    part = (1 + fit_error(a) + 2 * U) * (1 + rounding(dtype)) - 1
    assert (y < 0).all() and ((y.double() - want).abs() <= part * want.abs()).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_tail_of_the_slope(c8, dtype, kind):
    """t = Phi(-a) - a phi(a) from a = 1.5 on.  Of a phi(a) + Phi(-a), which is at most (1 + 2 / a^2) |t| / (1 - 1 / a^2): phi by 2^-22 of the
    exponential and the rounding of its argument, (0.73 a^2 + 1.4) log(2) twice U; Phi(-a), which is at most a phi(a) / a^2, by its fit;
    three roundings.  Where the sum's factor is taken as 1 / (1 - 1 / a^2)^2, the second order is in it too."""
    x = -torch.linspace(1.5, 12.9, 400001, device="cuda").to(dtype).view(-1, 1)
    kept = c8.pack8(x, kind)
    v = -kept.expand(F32).double()
    gx = c8.gelu8_backward(torch.ones_like(x), kept).double()
    there = (v >= 1.5) & (v <= 12.9)
    v, gx = v[there], gx[there]
    want = tail(v) - v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    part = (fit_error(v) / v ** 2 + 2.0 ** -22 + (0.73 * v ** 2 + 1.4) * math.log(2) * 2 * U + 3 * U) / (1 - 1 / v ** 2) ** 2
    part = (1 + part) * (1 + rounding(dtype)) - 1
    assert v.numel() > 1000 and ((gx - want).abs() <= part * want.abs()).all()


@pytest.mark.parametrize("dtype", [F32, torch.float16, BF16])
def test_absolute_bounds(c8, dtype):
    """What include/bsrl.h promises everywhere: 1e-7 + U |y| and 3e-7, then the type's rounding (half of its smallest step near zero)."""
    f = torch.finfo(dtype)
    x = torch.linspace(-14, 14, 400001, device="cuda").to(dtype).view(-1, 1)
    y, kept = c8.gelu8_forward(x)
    a = x.double()
    want = a * tail(-a)
    step = f.smallest_normal * f.eps / 2
    assert ((y.double() - want).abs() <= (want.abs() * (1 + U) + 1e-7) * (1 + f.eps / 2) - want.abs() + step).all()
    v = kept.expand(F32).double()
    slope = tail(-v) + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    gx = c8.gelu8_backward(torch.ones_like(x), kept).double()
    assert ((gx - slope).abs() <= (slope.abs() + 3e-7) * (1 + f.eps / 2) - slope.abs() + step).all()
