"""The bounds for gradients in two 16-bit parts tell them from one part: on the
CPU, results without the second part are outside."""
import pytest
import torch

import ffn_reference as ref
import ffn_two_parts as parts


def outside(got, want, t=None):
    value, bound = want if t is None else ref.rounded(*want, t)
    return ((got - value).abs() > bound).double().mean().item()


@pytest.mark.parametrize("t", parts.HALVES)
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("m,k,n", parts.SIZES)
def test_weight_gradient_beside_8_bits(t, act, m, k, n):
    x, w, b, dy = parts.linear_inputs(m, k, n, t)
    want = parts.linear_grads(x, w, b, dy, act)
    one = parts.linear_grads(x, w, b, dy, act, lo=False)
    assert outside(want[0][0].to(t).double(), want[0], t) == 0
    assert outside(one[0][0].to(t).double(), want[0], t) > 0.01


@pytest.mark.parametrize("t", parts.HALVES)
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("rows,d,h", parts.BLOCKS)
def test_norm_gradients_of_the_block(t, act, rows, d, h):
    args = parts.block_inputs(rows, d, h, t)
    x, nw, nb, w1, b1, w2, b2 = map(ref.wide, args)
    dy = parts.normal(rows, d, t=t, seed=9, scale=0.25)
    hid = ref.norm(x, nw, nb, 1e-5, t)[0][0].to(t).double()
    da = (ref.wide(dy) @ w2).to(t)
    given = (args[0], args[1], args[3], args[4], hid.to(t), da, dy, act)
    want, one = parts.norm_grads(*given), parts.norm_grads(*given, lo=False)
    dx = one[0][0].to(t).double()
    # sums over many rows have wider bounds
    if rows < 100:
        assert outside(one[2][0], want[2]) > 0.1
        assert outside(one[1][0], want[1]) > 0.05
        # of one row dw1 is a product that rounds once or twice
        dw1 = one[3][0].to(t).double()
        assert outside(dw1, want[3], t) > 0.02
    # one row has few values
    assert rows == 1 or outside(dx, want[0], t) > 0.02
