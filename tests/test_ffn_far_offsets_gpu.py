"""Rows whose place needs more than 32 bits, value by value."""
import pytest
import torch

import ffn_reference as ref
import gtopkssgd_amd as gt

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF = torch.bfloat16


def test_linear_layer_of_far_rows():
    rows, k, n = 300_000, 8192, 8
    at = torch.tensor([0, 131_072, 262_143, 262_145, rows - 1], device=DEV)
    g = torch.Generator().manual_seed(0)
    part = torch.randn(5, k, generator=g).to(BF).to(DEV)
    w = (torch.randn(n, k, generator=g) * 0.01).to(BF).to(DEV)
    x = torch.zeros(rows, k, device=DEV, dtype=BF)
    x[at] = part
    dy = torch.zeros(rows, n, device=DEV, dtype=BF)
    dy[at] = torch.randn(5, n, generator=g).to(BF).to(DEV)
    x.requires_grad_(True)
    y = gt.linear_act(x, w)
    dx, = torch.autograd.grad(y, x, dy)
    want = ref.linear(ref.wide(part), ref.wide(w), None, None, "none", BF,
                      dy=ref.wide(dy[at]))
    ref.close(y[at], *want[0], what="y")
    ref.close(dx[at], *want[1], what="dx")
    others = torch.ones(rows, dtype=torch.bool, device=DEV)
    others[at] = False
    assert not bool(y.detach()[others].any())
    # sums over few columns: the large matrix is not copied for this
    assert float(dx.abs().sum(1, dtype=torch.float32)[others].amax()) == 0
