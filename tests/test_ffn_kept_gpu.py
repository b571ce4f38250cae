"""What is kept of the value before gelu and silu has more bits than the result:
its slope is right to more than the result's own rounding."""
import pytest
import torch

import ffn_reference as ref
import gtopkssgd_amd as gt

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16
# half a step of what u is kept in
KEPT = {BF: ref.U[HF], HF: ref.E}


def inputs(m, k, n, t):
    """u in steps of 2^-13 up to some 4: exact in fp32 in any order of summing,
    with more bits than either 16-bit type has."""
    g = torch.Generator().manual_seed(m + k + n)
    x = torch.randint(-4, 5, (m, k), generator=g) * 2.0 ** -6
    w = torch.randint(-16, 17, (n, k), generator=g) * 2.0 ** -7
    b = torch.randint(-2 ** 15, 2 ** 15, (n,), generator=g) * 2.0 ** -13
    dy = torch.randn(m, n, generator=g)
    return x.to(t), w.to(t), b, dy.to(t)


@pytest.mark.parametrize("m,k,n", [(1, 30, 700), (40, 64, 300), (300, 33, 130),
                                   (900, 500, 70)])
@pytest.mark.parametrize("t", [BF, HF])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_slope_of_the_kept_value(m, k, n, t, act):
    """The bias's gradient in fp32 is the sum of dy slope(u) without a rounding
    to the type; of one row it is each of them."""
    x, w, b, dy = (v.to(DEV) for v in inputs(m, k, n, t))
    b.requires_grad_(True)
    db, = torch.autograd.grad(gt.linear_act(x, w, b, act=act), b, dy)
    u = ref.wide(x) @ ref.wide(w).t() + ref.wide(b)
    assert torch.equal(u, u.float().double())
    d = ref.wide(dy)
    s = ref.slope(u, act)
    off = d.abs() * (ref.CURVE * KEPT[t] * u.abs() + ref.FUNC * (1 + u.abs())) \
        + 4 * ref.E * (d * s).abs()
    ref.close(db, (d * s).sum(0), off.sum(0) +
              (m + 8) * ref.E * (d * s).abs().sum(0), what="db")


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("rows", [3, 100])
def test_values_beyond_fp16(act, rows):
    """Beside bf16, u past fp16's largest value: the slope is 0 or 1."""
    big = torch.tensor([7e4, -7e4, 1e30, -1e30, 65504.0, -65504.0, 1e-30, 0.0],
                       device=DEV).to(BF)
    x = big.repeat(rows)[:, None].requires_grad_(True)
    y = gt.linear_act(x, torch.ones(1, 1, device=DEV, dtype=BF), act=act)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    want = torch.tensor([1, 0, 1, 0, 1, 0, 0.5, 0.5], dtype=BF, device=DEV)
    assert torch.equal(dx[:, 0], want.repeat(rows))
