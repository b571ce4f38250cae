"""Layer norm's gradients where rows lie far from zero for their spread.

The values are small multiples of powers of two, so that their sums, their mean
and their variance come out exact in fp32: what is left of x - mean has no
rounding, and xh is off by a few steps of itself, not of x."""
import pytest
import torch

import ffn_reference as ref
import gtopkssgd_amd as gt

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
E = ref.E


def normal(*shape, t=FP, seed=0, shift=0.0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return (torch.randn(*shape, generator=g) + shift).to(t).to(DEV)


def want_grads(x, w, dy, kept, eps):
    """dx and dweight in 64 bits with bounds; mean and variance are exact."""
    n = x.shape[1]
    mean = x.mean(1, keepdim=True)
    # 64 bits round, too: the mean without what that leaves is the exact one
    mean = mean + (x - mean).mean(1, keepdim=True)
    var = (x - mean).square().mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    # 1 / sqrt(v + eps): eps, the sum, the root and the quotient round
    dr = 4 * E
    hat = (kept - mean) * rstd
    # kept - mean rounds once, its product once, and rstd as above
    dhat = (2 * E + dr) * hat.abs()
    g = dy * w
    m1, m2 = g.mean(1, keepdim=True), (g * hat).mean(1, keepdim=True)
    dm1 = (n + 8) * E * g.abs().mean(1, keepdim=True)
    dm2 = (n + 8) * E * (g * hat).abs().mean(1, keepdim=True) + \
        (g.abs() * dhat).mean(1, keepdim=True)
    dx = rstd * (g - m1 - hat * m2)
    bound = dm1 + dm2 * hat.abs() + dhat * (m2.abs() + dm2) + \
        8 * E * (g.abs() + m1.abs() + (hat * m2).abs())
    rows = x.shape[0]
    return ((dx, bound * rstd + dr * dx.abs()),
            ((dy * hat).sum(0), (dy.abs() * dhat).sum(0) +
             (rows + 8) * E * (dy * hat).abs().sum(0)))


def check(x, act8, eps=1e-5):
    t, n = x.dtype, x.shape[1]
    x.requires_grad_(True)
    w = normal(n, seed=1, shift=1.0).requires_grad_(True)
    dy = normal(*x.shape, t=t, seed=2)
    y = gt.layer_norm(x, w, None, eps, act8=act8)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    wide = ref.wide(x)
    kept = ref.pack_values(wide) if act8 else wide
    want = want_grads(wide, ref.wide(w), ref.wide(dy), kept, eps)
    ref.close(dx, *ref.rounded(*want[0], t), what="dx")
    ref.close(dw, *ref.rounded(*want[1], FP), what="dweight")
    return dw


@pytest.mark.parametrize("dim", [7, 100, 1000, 1500, 2048])
@pytest.mark.parametrize("t,value", [
    (FP, 1000.0), (FP, 4097.0), (FP, 123456.0), (BF, 1000.0), (BF, 4128.0),
    (BF, 123392.0), (HF, 1000.0), (HF, 4100.0)])
@pytest.mark.parametrize("act8", [False, True])
def test_rows_of_one_value(dim, t, value, act8):
    """xh is 0: nothing of dy gets into dweight, and dx is rstd (g - mean g)."""
    x = torch.full((6, dim), value, dtype=t, device=DEV)
    assert (x == value).all()
    dw = check(x, act8)
    if not act8:
        assert (dw == 0).all()


@pytest.mark.parametrize("dim", [4096, 8192, 16384, 32768, 40000])
@pytest.mark.parametrize("act8", [False, True])
def test_long_rows_of_one_value(dim, act8):
    dw = check(torch.full((3, dim), 1000.0, device=DEV), act8)
    if not act8:
        assert (dw == 0).all()


@pytest.mark.parametrize("dim", [8, 64, 200, 1024, 1500, 4000])
@pytest.mark.parametrize("t,centre,step", [
    (FP, 1000.0, 1.0), (FP, -4097.0, 1.0), (FP, 2.0, 2.0 ** -10),
    (BF, 136.0, 1.0), (HF, 1025.0, 1.0)])
@pytest.mark.parametrize("act8", [False, True])
def test_small_spread_round_a_large_mean(dim, t, centre, step, act8):
    """Half of a row's values lie as far above the centre as the others below
    it: the mean is the centre, the squares' sum a whole number of steps."""
    g = torch.Generator().manual_seed(dim)
    off = torch.randint(0, 4, (5, dim // 2), generator=g).float() * step
    off = torch.cat([off, -off], 1)[:, torch.randperm(dim, generator=g)]
    x = (centre + off).to(t).to(DEV)
    assert torch.equal(x.cpu().double(), centre + off.double())
    check(x, act8)
