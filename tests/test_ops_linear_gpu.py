"""Linear layers on compressed weights far from zero: gradients of units that an activation has nearly
closed, against their formula in 64 bits."""

import pytest
import torch

import cuzipnn_b200 as z
from test_ops_gpu import ACTS, BF, DEV, HF, assert_within, rnd, sum_bound, u_of, weight

pytestmark = pytest.mark.gpu


def closed_units(act, at, dtype, tokens, rows, cols=64):
    """(dbias, its formula, the bound): all units have a z near `at`, where the derivative is small.

    The derivative is kept to 2^-11 of itself and evaluated to 2^-16; it changes by 2 + |z| of itself
    per unit of z (gelu's tail falls like exp(-z^2 / 2), silu's like exp(z)), z being off by its sum's
    bound.  Sums are in 32 bits, the result is rounded once."""
    w, blob = weight(rows, cols, dtype)
    x = rnd(tokens, cols, dtype=dtype, scale=0.25)
    bias = (at + 0.01 * torch.arange(rows, device=DEV) / rows).to(dtype).requires_grad_()
    g = rnd(tokens, rows, dtype=dtype, seed=5).abs() + 0.5
    gain = 2.0**-round(torch.log2(act_slope(act, torch.tensor([at], device=DEV, dtype=torch.double)).abs()).item())
    if dtype == BF:
        g = (g * gain).to(dtype)  # bf16 has the range for it
    db, = torch.autograd.grad(z.blob_linear(x, blob, bias=bias, activation=act), [bias], g)
    zz = x.double() @ w.double().t() + bias.detach().double()
    slope = act_slope(act, zz)
    ez = sum_bound(cols) * (x.double().abs() @ w.double().abs().t() + bias.detach().double().abs())
    want = (slope * g.double()).sum(0)
    mass = ((2.0**-11 + 2.0**-16 + (2 + zz.abs()) * ez) * slope.abs() * g.double()).sum(0)
    mass = mass + (2.0**-40 * g.double()).sum(0) + sum_bound(tokens) * (slope.abs() * g.double()).sum(0)
    return db, want, mass + u_of(dtype) * want.abs() + (2.0**-25 if dtype == HF else 0.0)


def act_slope(act, zz):
    zz = zz.detach().clone().requires_grad_()
    return torch.autograd.grad(ACTS[act](zz).sum(), zz)[0]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("act,at", [("silu", -6.0), ("silu", -8.0), ("silu", -10.0), ("gelu_tanh", -3.5), ("gelu", -3.25)])
@pytest.mark.parametrize("tokens,rows", [(1, 64), (40, 333), (600, 264)])
def test_bias_gradient_of_closed_units(act, at, tokens, rows, dtype):
    assert_within(*closed_units(act, at, dtype, tokens, rows))


def test_bias_gradient_of_far_units():
    """Further out, where bf16 holds the gradient and fixed point held nothing."""
    for act, at in (("silu", -14.0), ("silu", -18.0), ("gelu_tanh", -4.5)):
        db, want, bound = closed_units(act, at, BF, 200, 256)
        assert_within(db, want, bound)
        assert bool((want.abs() > 8 * bound).all())  # (the bound says something)


@pytest.mark.parametrize("at", [-4.0, -5.0, -5.5])
@pytest.mark.parametrize("tokens", [1, 200])
def test_bias_gradient_of_units_far_below_gelus_zero(tokens, at):
    db, want, bound = closed_units("gelu", at, BF, tokens, 256)
    assert_within(db, want, bound)
    assert bool((want.abs() > 4 * bound).all())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("act,at", [("gelu", -3.0), ("gelu", -4.5), ("gelu", -6.0), ("gelu_tanh", -4.0), ("silu", -9.0),
                                    ("gelu", 0.0), ("gelu", 2.0)])
@pytest.mark.parametrize("tokens,rows", [(1, 64), (40, 333)])
def test_values_of_closed_units(act, at, tokens, rows, dtype):
    """act(z) is off by 2^-16 of itself, by z's error (as its derivative) and by one rounding."""
    w, blob = weight(rows, 64, dtype)
    x = rnd(tokens, 64, dtype=dtype, scale=0.25)
    bias = (at + 0.5 * torch.linspace(-1, 1, rows, device=DEV)).to(dtype)
    y = z.blob_linear(x, blob, bias=bias, activation=act)
    zz = x.double() @ w.double().t() + bias.double()
    want = ACTS[act](zz)
    if act == "gelu":  # 1 + erf loses digits in 64 bits too
        want = zz * 0.5 * torch.special.erfc(-zz * 0.5**0.5)
    ez = sum_bound(64) * (x.double().abs() @ w.double().abs().t() + bias.double().abs())
    bound = (2.0**-16 + u_of(dtype)) * want.abs() + 1.05 * ez * act_slope(act, zz).abs() + 2.0 * ez * ez
    assert_within(y, want, bound + (2.0**-25 if dtype == HF else 0.0))
