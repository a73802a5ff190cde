"""The derivatives of the dense layers' activations, one by one: with the identity for a weight z is x and dx is
d = g f'(z), so that nothing is summed and each element has a bound of its own.

d is rounded to the type (u) and f' is kept in a form of its own beside the 16-bit types; f' itself is off by what its
formula makes of float32 steps (s = 2^-24): an exponential of argument a by 1.5 |a| s (the rounded argument and the
constant in it) and two s of its own, a reciprocal by two."""
import math

import pytest
import torch

import xnn_amd as xa

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
S = 2.0 ** -24


def _formula(name, z):
    """f'(z) in float64 and the relative error of its evaluation."""
    a = z.abs()
    if name == "silu":
        p = torch.sigmoid(z)
        slope = p * (1 + z * torch.sigmoid(-z))
        # p; and 1 + z (1 - p), whose terms are of size |z| and 1
        return slope, (1.5 * a + 8) * S + p * (a + 2) * 8 * S / slope.abs().clamp_min(1e-300)
    if name == "tanh":
        e = torch.exp(-2 * a)
        return 4 * e / (1 + e) ** 2, (3 * a + 12) * S
    phi = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2))
    slope = z * phi + cdf
    each = (a * phi + cdf) / slope.abs().clamp_min(1e-300)
    return slope, each * (1.5 * z * z + 16) * S


def _five_terms(z):
    """By how much the five-term formula of the 16-bit types is off in Phi(z) (Abramowitz and Stegun 7.1.26)."""
    x = z.abs() / math.sqrt(2)
    t = 1 / (1 + 0.3275911 * x)
    q = 0.0
    for c in (1.061405429, -1.453152027, 1.421413741, -0.284496736, 0.254829592):
        q = (q + c) * t
    return (q * torch.exp(-x * x) - torch.special.erfc(x)).abs() / 2


def _kept(dtype, slope):
    """By how much f' is off as it is kept."""
    a = slope.abs()
    if dtype == "f32":
        return torch.zeros_like(a)
    if dtype == "bf16":
        return 2.0 ** -11 * a + 2.0 ** -40
    # its root in steps of 1 / 30,000 from 2^-7 on, below it in float16 of 2^5 times it
    root = (2 * a.sqrt() / 60000 + 60000.0 ** -2) * 1.01
    return torch.where(a >= 2.0 ** -7, root, 2.0 ** -11 * a + 2.0 ** -30)


def _check(dtype, name, z, width, scale):
    """z, any number of values, in rows of `width`."""
    t = TYPES[dtype]
    z = z.to(t)
    z = torch.cat([z, z[:1].expand(-len(z) % width)]).view(-1, width).to(DEV)
    gen = torch.Generator().manual_seed(width)
    g = (torch.randn(z.shape, generator=gen) * scale).to(t).to(DEV)
    leaf = z.clone().requires_grad_(True)
    out = xa.linear(leaf, torch.eye(width, dtype=t, device=DEV), None, name)
    got, = torch.autograd.grad(out, leaf, g)
    slope, off = _formula(name, z.double())
    if name == "gelu" and dtype != "f32":
        off = off + _five_terms(z.double()) / slope.abs()
    u = torch.finfo(t).eps / 2
    d = g.double() * slope
    kept = _kept(dtype, slope)
    bound = (d.abs() * off + g.double().abs() * kept) * (1 + u) + u * d.abs() + (2.0 ** -126 if dtype == "f32" else 2.0 ** -25)
    err = (got.double() - d).abs()
    worst = int((err / bound).argmax())
    assert got.isfinite().all() and float(err.flatten()[worst]) <= float(bound.flatten()[worst]), (
        float(z.flatten()[worst]), float(err.flatten()[worst] / d.abs().flatten()[worst]),
        float(err.flatten()[worst] / bound.flatten()[worst]))


TAILS = {"silu": (-14.0, -6.0), "tanh": (3.0, 7.0), "gelu": (-5.0, -2.5)}


# d is formed as the products stage it, and by a pass of its own; the cotangents as small as they come, and as a loss
# scale has them
def _check_tail(dtype, name):
    lo, hi = TAILS[name]
    z = torch.linspace(lo, hi, 4000)
    for width in (64, 192):
        for scale in (1.0, 1024.0):
            _check(dtype, name, z, width, scale)
            if name == "tanh":
                _check(dtype, name, -z, width, scale)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_tanh_far_from_zero(dtype):
    """f' is 4 e / (1 + e)^2, e = exp(-2 |z|): 1 - y^2 has lost it where y is near 1."""
    _check_tail(dtype, "tanh")


@pytest.mark.parametrize("name", TAILS)
def test_float16_far_from_one(name):
    """Small f' keep the type's digits: a loss scale makes their gradients large."""
    _check_tail("f16", name)


@pytest.mark.parametrize("name", TAILS)
def test_every_slope_of_float16_as_it_is_kept(name):
    """Over the whole range, the largest and the least among them: 1.13 and -0.13 of gelu at -+1.414, zeros, and the
    borders between the forms."""
    z = torch.cat([torch.linspace(-20, 20, 20001), torch.linspace(-1.5, -1.2, 2000), torch.linspace(1.3, 2.5, 2000),
                   torch.linspace(3.0, 3.2, 500), torch.zeros(3)])
    for width in (64, 192):
        _check("f16", name, z, width, 1.0)


def test_slopes_that_are_not_numbers_stay_so():
    for dtype, t in TYPES.items():
        for width in (64, 192):
            x = torch.randn(40, width, generator=torch.Generator().manual_seed(1)).to(t).to(DEV)
            x[3] = float("nan")
            leaf = x.clone().requires_grad_(True)
            out = xa.linear(leaf, torch.eye(width, dtype=t, device=DEV), None, "tanh")
            got, = torch.autograd.grad(out, leaf, torch.ones_like(out))
            assert got[3].isnan().all() and got[:3].isfinite().all() and got[4:].isfinite().all()


def test_gelu_in_float32():
    """Output and slope, z being x exactly, in steps s = 2^-24 of the result. Below -1: the exponential's 1.25 z^2 (its
    argument z^2 / 2 has two roundings and a constant, 2.5 s) and two, t's three, the polynomial's six, three products.
    In (-1, 0) Phi(z), above 0.158, is off by 0.75 s, five of its own; in (0, 1) it is above 1/2 and off by 1.2 s; from 1
    on by 15 s of q < 0.159 and half a step, above 0.84. The last product adds one."""
    z = torch.cat([torch.linspace(-9, 9, 60001), torch.linspace(-1.01, -0.99, 1001), torch.linspace(0.99, 1.01, 1001),
                   torch.logspace(-30, 0, 2000), -torch.logspace(-30, 0, 2000)])
    for width in (64, 192):
        _check("f32", "gelu", z, width, 1.0)
    x = torch.cat([z, z[:1].expand(-len(z) % 64)]).view(-1, 64).to(DEV)
    got = xa.linear(x, torch.eye(64, device=DEV), None, "gelu").double()
    x = x.double()
    want = x * 0.5 * torch.special.erfc(-x / math.sqrt(2))
    steps = torch.where(x > -1, 4 + 4 * (x < 0) + 2 * (x >= 1), 1.25 * x * x + 16) * S
    err = (got - want).abs() / (steps * want.abs()).clamp_min(2.0 ** -149)
    assert float(err.max()) <= 1.0, float(x.flatten()[err.argmax()])
