"""Inputs and 64-bit results with bounds for gradients that are kept in two
16-bit parts.  ``lo=False``: what comes out where the second part is dropped."""
import torch

import ffn_reference as ref

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
HALVES = [BF, HF]
E, U = ref.E, ref.U
# odd numbers of rows, sums in one part and in several, one and more tiles
SIZES = [(70, 40, 24), (131, 129, 77), (1500, 200, 130), (3001, 130, 65)]
BLOCKS = [(1, 40, 100), (37, 101, 403), (221, 130, 1000), (700, 65, 257)]


TERMS = 30     # of a sum that are not 0: adding a 0 does not round


def sparse(v, among, seed=0):
    """TERMS of `among` values stay on the average"""
    g = torch.Generator().manual_seed(seed + sum(v.shape))
    return v * (torch.rand(v.shape, generator=g) < TERMS / among)


def summed(a, b, da, parts):
    """a @ b in fp32 with a off by da, and the bound; each value of a is the sum
    of so many parts."""
    terms = parts * ((a != 0).double() @ (b != 0).double())
    return a @ b, (terms + 8) * E * (a.abs() @ b.abs()) + da @ b.abs()


def rounded_to(v, off, t):
    """v, off by `off`, rounded: to one value, but for those within their error
    of a border"""
    low, high = (v - off).to(t).double(), (v + off).to(t).double()
    return (low + high) / 2, (high - low) / 2


def normal(*shape, t=FP, seed=0, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return (torch.randn(*shape, generator=g) * scale + shift).to(t)


# ---- the weight's gradient beside x in 8 bits ----------------------------------

def linear_inputs(m, k, n, t):
    """x of -1, 0 and 1: its 8-bit form is itself.  w and b in steps of 2^-4:
    u has no rounding in any order."""
    g = torch.Generator().manual_seed(m + k + n)
    x = sparse(torch.randint(0, 2, (m, k), generator=g) * 2.0 - 1, m)
    w = torch.randint(-4, 5, (n, k), generator=g) * 2.0 ** -4
    b = torch.randint(-16, 17, (n,), generator=g) * 2.0 ** -3
    return x.to(t), w.to(t), b.to(t), normal(m, n, t=t, seed=4)


def p_of(dy, u, act, t, lo):
    """dy act'(u) with its error, u exact."""
    s = ref.slope(u, act)
    p = dy * s
    off = dy.abs() * ref.FUNC * (1 + u.abs()) + 4 * E * p.abs()
    if lo:
        return p, off + U[t] ** 2 * p.abs() + ref.TINY[t]
    hi = p.to(t).double()
    return hi, off


def linear_grads(x, w, b, dy, act, lo=True):
    """[dw, db] with bounds, where two parts are multiplied; or what dropping
    one gives, with the same bounds"""
    t = x.dtype
    x, w, b, dy = map(ref.wide, (x, w, b, dy))
    assert torch.equal(ref.pack_values(x).float().double(), x)
    u = ref.pack_values(x @ w.t() + b)
    whole, dp = p_of(dy, u, act, t, True)
    p = whole if lo else p_of(dy, u, act, t, False)[0]
    m = x.shape[0]
    return ((p.t() @ x, summed(whole.t(), x, dp.t(), 2)[1]),
            (whole.sum(0), dp.sum(0) + (m + 8) * E * whole.abs().sum(0)))


# ---- the norm's gradients in the block -----------------------------------------------

def block_inputs(rows, d, h, t):
    """the norm's parameters in fp32, whose gradients are not rounded further"""
    return [normal(rows, d, t=t),
            normal(d, scale=0.2, shift=1.0, seed=1), normal(d, seed=2),
            sparse(normal(h, d, t=t, seed=3), h),
            normal(h, t=t, scale=0.1, seed=4),
            normal(d, h, t=t, scale=h ** -0.5, seed=5), normal(d, t=t, seed=6)]


def norm_grads(x, nw, w1, b1, hid, da, dy, act, lo=True):
    """[dx, dweight, dbias] of the norm, dy onto dx, and dw1, from the rounded hid
    and da."""
    t = x.dtype
    x, nw, w1, b1, hid, da, dy = map(ref.wide, (x, nw, w1, b1, hid, da, dy))
    u, du = summed(hid, w1.t(), torch.zeros_like(hid), 1)
    u = u + b1
    u, du = rounded_to(u, du + 2 * E * b1.abs(), HF if t == BF else FP)
    whole, dp = p_of(da, u, act, t, True)
    dp = dp + ref.CURVE * du * da.abs()
    p = whole if lo else p_of(da, u, act, t, False)[0]
    v, bound = summed(whole, w1, dp, 2)
    dh, ddh = rounded_to(v, bound, t)
    if not lo:
        dh = (p @ w1).to(t).double()
    dx, dw, db = ref.norm(x, nw, None, 1e-5, t, dy=dh)[1:]
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    rstd = 1 / torch.sqrt(var + 1e-5)
    hat = (x - mean) * rstd
    g = ddh * nw.abs()
    off = rstd * (g + g.mean(1, keepdim=True) +
                  hat.abs() * (g * hat.abs()).mean(1, keepdim=True))
    return ((dx[0] + dy, dx[1] + off + E * (dx[0].abs() + dy.abs())),
            (dw[0], dw[1] + (ddh * hat.abs()).sum(0)),
            (db[0], db[1] + ddh.sum(0)),
            (p.t() @ hid, summed(whole.t(), hid, dp.t(), 2)[1]))
