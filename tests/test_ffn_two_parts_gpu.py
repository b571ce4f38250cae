"""The second part of a gradient that is kept in two 16-bit parts: bounds under
what the result would be off by without it (tests/test_ffn_two_parts.py shows
that on the CPU)."""
import pytest
import torch

import ffn_reference as ref
import ffn_two_parts as parts
import gtopkssgd_amd as gt

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("t", parts.HALVES)
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("m,k,n", parts.SIZES)
def test_weight_gradient_beside_8_bits(t, act, m, k, n):
    x, w, b, dy = (v.to(DEV) for v in parts.linear_inputs(m, k, n, t))
    leaves = [w.requires_grad_(True), b.requires_grad_(True)]
    y = gt.linear_act(x, *leaves, act=act, act8=True)
    dw, db = torch.autograd.grad(y, leaves, dy)
    want = parts.linear_grads(x, w, b, dy, act)
    ref.close(dw, *ref.rounded(*want[0], t), what="dw")
    ref.close(db, *ref.rounded(*want[1], t), what="db")


@pytest.mark.parametrize("t", parts.HALVES)
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("rows,d,h", parts.BLOCKS)
def test_norm_gradients_of_the_block(t, act, rows, d, h):
    """dh from two parts of p: its sum over the rows is the norm bias's gradient,
    which fp32 keeps, and dx and the norm weight's are made from it.  What the
    block keeps on its way is taken from the operators themselves, which give
    the same bits."""
    args = [v.to(DEV).requires_grad_(True)
            for v in parts.block_inputs(rows, d, h, t)]
    dy = parts.normal(rows, d, t=t, seed=9, scale=0.25).to(DEV)
    x, nw, nb, w1, b1, w2, b2 = args
    with torch.no_grad():
        hid = gt.layer_norm(x, nw, nb)
        a = gt.linear_act(hid, w1, b1, act=act)
    a.requires_grad_(True)
    da, = torch.autograd.grad(gt.linear_act(a, w2, b2, x), a, dy)
    got = torch.autograd.grad(gt.ffn_block(*args, act=act), [x, nw, nb, w1],
                              dy)
    want = parts.norm_grads(x, nw, w1, b1, hid, da, dy, act)
    ref.close(got[2], *want[2], what="norm bias")
    ref.close(got[1], *want[1], what="norm weight")
    ref.close(got[0], *ref.rounded(*want[0], t), what="dx")
    ref.close(got[3], *ref.rounded(*want[3], t), what="dw1")
