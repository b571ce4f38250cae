"""gelu and its slope far below 0, where the value is a small one, relative to
itself: 64 bits against 16 bits, with one value a sum so that u is exact."""
import math

import pytest
import torch

import ffn_reference as ref
import gtopkssgd_amd as gt

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16


def cdf(v):
    """Phi(v), of which torch's ndtr keeps nothing under 1e-16"""
    return 0.5 * torch.erfc(-v * 0.5 ** 0.5)


def tail_off(v):
    """What the fast tail is off by, of itself: its fit 2^-16.2; the exponent
    0.72 v^2, three times rounded, which exp2 turns into 1.5 v^2 steps; the
    others 10."""
    return 2.0 ** -16.2 + (10 + 1.5 * v * v) * ref.E


def inputs(t, low, high):
    """every value of the type from low to high"""
    u = torch.arange(2 ** 15, dtype=torch.int16).view(t)
    u = u[torch.isfinite(u)]
    u = torch.cat([u, -u])
    return u[(u >= low) & (u <= high)].to(DEV)


@pytest.mark.parametrize("t,low", [(BF, -12.0), (HF, -5.5)])
@pytest.mark.parametrize("rows", [60, 400])
def test_gelu_by_relative_size(t, low, rows):
    """Up to 64 rows, and more of them, go to kernels of their own."""
    w = torch.ones(1, 1, device=DEV, dtype=t)
    for u in inputs(t, low, 12.0).split(rows):
        x = u[:, None].requires_grad_(True)
        y = gt.linear_act(x, w, act="gelu")
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        v = ref.wide(u)
        tail = cdf(-v.abs())
        want = v * cdf(v)
        # y = u - u q above 0, u q below
        ref.close(y[:, 0], *ref.rounded(
            want, v.abs() * tail * tail_off(v) + 4 * ref.E * want.abs(), t),
            what="gelu")
        edge = v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
        slope = cdf(v) + edge
        # Phi and u phi, off by the tail's error each, and by their sum's
        # rounding; p and dx are the same value in the type
        off = (tail + edge.abs()) * tail_off(v) + \
            4 * ref.E * (cdf(v) + edge.abs())
        ref.close(dx[:, 0], *ref.rounded(slope, off, t), what="slope")


@pytest.mark.parametrize("t", [BF, HF])
def test_gelu_beyond_the_tail(t):
    """Past it nothing is left below 0, and u itself above."""
    u = torch.tensor([-40.0, -1000.0, -float("inf"), 40.0, 1000.0,
                      float("inf")], device=DEV).to(t)
    x = u[:, None].requires_grad_(True)
    y = gt.linear_act(x, torch.ones(1, 1, device=DEV, dtype=t), act="gelu")
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert y[:, 0].tolist() == [0, 0, 0] + u[3:].tolist()
    assert dx[:, 0].tolist() == [0, 0, 0, 1, 1, 1]


def test_gelu_slope_in_32_bits():
    """Phi below 0 is the tail itself, not 1/2 less what is left of it."""
    u = -torch.linspace(0, 12, 4001, device=DEV)
    x = u[:, None].requires_grad_(True)
    y = gt.linear_act(x, torch.ones(1, 1, device=DEV), act="gelu")
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    v = ref.wide(u)
    edge = v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
    # erfc is off by 16 units at most, exp by fewer, and each by its argument's
    # rounding: v^2 / 2, of which the derivative makes as many steps
    rel = (40 + 2 * v * v) * ref.E
    ref.close(dx[:, 0], cdf(v) + edge, (cdf(v) + edge.abs()) * rel + 2.0 ** -126)
    ref.close(y[:, 0], v * cdf(v), (v * cdf(v)).abs() * rel + 2.0 ** -126)
