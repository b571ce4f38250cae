"""The feed-forward operators in 64 bits on the CPU, with bounds on how far a
16- or 32-bit result may be from them.

Each function returns (value, bound) pairs.  A bound counts, value by value:

* half a step of each rounding to the type: U[t] |value|, U = eps / 2;
* a sum of n fp32 terms: (n + 8) 2^-24 times the sum of the terms' sizes (the
  worst order of adding; 8 covers what surrounds the sum: bias, activation,
  residual, the product with a scale);
* an error of an operand times the other operand's size.

The functions exp, erf and their like are taken to be within 2^-20 of the
argument's size: the fast ones for 16 bits are within 1.5e-7 absolute.
"""
import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11,
     torch.float32: 2.0 ** -24}
E = 2.0 ** -24
FUNC = 2.0 ** -20
# below the smallest normal numbers a rounding is off by half the smallest step
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25,
        torch.float32: 2.0 ** -126}
GROUP = 128
# largest |act''|: gelu 2 phi(0), silu 1/2; largest |act'|: gelu 1.13, silu 1.1
CURVE, SLOPE = 0.8, 1.13


def wide(t):
    return None if t is None else t.detach().double().cpu()


def rounded(value, bound, t):
    return value, bound + U[t] * (value.abs() + bound) + TINY[t]


def pack_values(x):
    """What stands for x after 8 bits: fp32 steps, by definition."""
    x = x.float()
    rows, dim = x.shape
    out = torch.empty(rows, dim, dtype=torch.double)
    for g in range(0, dim, GROUP):
        part = x[:, g:g + GROUP]
        a = part.abs().amax(1, keepdim=True)
        some = a >= 2.0 ** -119
        by = torch.where(some, torch.full_like(a, 127.0) / a, 0 * a)
        s = torch.where(some, a * torch.full_like(a, 1.0 / 127.0), 0 * a)
        out[:, g:g + GROUP] = torch.round(part * by).double() * s.double()
    return out


def act(u, name):
    if name == "relu":
        return u.clamp_min(0)
    if name == "gelu":
        return u * torch.special.ndtr(u)
    if name == "silu":
        return u * torch.sigmoid(u)
    return u


def slope(u, name):
    if name == "none":
        return torch.ones_like(u)
    if name == "relu":
        return (u > 0).double()
    if name == "gelu":
        return torch.special.ndtr(u) + \
            u * torch.exp(-0.5 * u * u) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(u)
    return s * (1 + u * (1 - s))


def mm(a, b, da=None, db=None):
    """a @ b, off by da and db in the operands, summed in fp32."""
    size = a.abs() @ b.abs()
    bound = (a.shape[1] + 8) * E * size
    if da is not None:
        bound = bound + da @ b.abs()
    if db is not None:
        bound = bound + a.abs() @ db
    return a @ b, bound


def norm(x, w, b, eps, t, act8=False, dy=None, kept=None):
    """[y, dx, dw, db] with bounds; dx etc. where dy is given."""
    n = x.shape[1]
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    one = torch.ones(n, dtype=torch.double)
    w1 = one if w is None else w
    hat = (x - mean) * rstd
    # mean and each x - mean are off by a few steps of the largest term, the
    # deviation's sum by n steps of itself
    top = x.abs().amax(1, keepdim=True)
    dmean = (n + 8) * E * x.abs().mean(1, keepdim=True)
    dhat = (dmean + 2 * E * top) * rstd + \
        hat.abs() * ((n + 8) * E + (dmean * rstd) ** 2)
    y = hat * w1 + (0 if b is None else b)
    ybound = dhat * w1.abs() + 4 * E * (hat.abs() * w1.abs() + y.abs())
    out = [rounded(y, ybound, t)]
    if dy is None:
        return out
    k = x if kept is None else kept
    hat = (k - mean) * rstd
    dhat = (dmean + 2 * E * (top + k.abs())) * rstd + \
        hat.abs() * ((n + 8) * E + (dmean * rstd) ** 2)
    g = dy * w1
    m1, m2 = g.mean(1, keepdim=True), (g * hat).mean(1, keepdim=True)
    dm1 = (n + 8) * E * g.abs().mean(1, keepdim=True)
    dm2 = (n + 8) * E * (g * hat).abs().mean(1, keepdim=True) + \
        (g.abs() * dhat).mean(1, keepdim=True)
    inner = g - m1 - hat * m2
    ibound = dm1 + dm2 * hat.abs() + dhat * (m2.abs() + dm2) + \
        8 * E * (g.abs() + m1.abs() + (hat * m2).abs())
    dx = rstd * inner
    out.append((dx, ibound * rstd + dx.abs() * ((n + 8) * E +
                                                (dmean * rstd) ** 2)))
    rows = x.shape[0]
    out.append(((dy * hat).sum(0),
                (dy.abs() * dhat).sum(0) +
                (rows + 8) * E * (dy * hat).abs().sum(0)))
    out.append((dy.sum(0), (rows + 8) * E * dy.abs().sum(0)))
    return out


def through(dy, ddy, u, du, name, t, act8, split):
    """p = dy act'(u) as the products are given it."""
    if name == "none":
        return dy, ddy
    if name == "relu":  # within its error of 0, u may fall on either side
        at_edge = (u.abs() <= du).double()
        return dy * slope(u, name), ddy + dy.abs() * at_edge
    if act8:
        u, du = pack_values(u), torch.zeros_like(u)
    else:
        du = du + U[t] * (u.abs() + du) + TINY[t]
    s = slope(u, name)
    p = dy * s
    bound = ddy * (s.abs() + FUNC * (1 + u.abs())) + \
        (dy.abs() + ddy) * (CURVE * du + FUNC * (1 + u.abs())) + 4 * E * p.abs()
    if split:  # what rounding leaves is kept, and rounds itself
        return p, bound + U[t] ** 2 * p.abs() + TINY[t]
    return p, bound + U[t] * (p.abs() + bound) + TINY[t]


def linear(x, w, b, res, name, t, act8=False, dy=None):
    """[y, dx, dw, db] with bounds."""
    u, du = mm(x, w.t())
    if b is not None:
        u = u + b
        du = du + 2 * E * b.abs()
    y = act(u, name)
    bound = SLOPE * du + FUNC * (u.abs() if name in ("gelu", "silu") else 0)
    if res is not None:
        y = y + res
        bound = bound + 2 * E * (y.abs() + res.abs())
    out = [rounded(y, bound, t)]
    if dy is None:
        return out
    split = act8 and t != torch.float32
    zero = torch.zeros_like(dy)
    p, dp = through(dy, zero, u, du, name, t, act8, False)
    dx, bx = mm(p, w, dp)
    out.append(rounded(dx, bx, t))
    p, dp = through(dy, zero, u, du, name, t, act8, split)
    k = pack_values(x) if act8 else x
    dk = U[t] * k.abs() + TINY[t] if act8 else torch.zeros_like(k)
    dw, bw = mm(p.t(), k, dp.t(), dk)
    out.append(rounded(dw, bw, t))
    # the bias's gradient is summed before p is rounded
    p, dp = through(dy, zero, u, du, name, t, act8, True)
    out.append((p.sum(0), dp.sum(0) + (p.shape[0] + 8) * E * p.abs().sum(0)))
    return out


def close(got, want, bound, what=""):
    got = got.detach().double().cpu().reshape(want.shape)
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst "
        f"{(off / bound.clamp_min(1e-300)).max().item():.3g} times the bound "
        f"at {divmod(int((off / bound.clamp_min(1e-300)).argmax()), want.shape[-1] if want.dim() else 1)}: "
        f"got {got.flatten()[int((off / bound.clamp_min(1e-300)).argmax())]:.8g}"
        f", want {want.flatten()[int((off / bound.clamp_min(1e-300)).argmax())]:.8g}")
