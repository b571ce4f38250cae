"""Results of the feed-forward operators may be modified in place, as those of
torch's own layers may."""
import pytest
import torch
import torch.nn.functional as F

import gtopkssgd_amd as gt

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
NAMES = ["norm", "norm8", "linear", "gelu8", "block", "block8"]
SHAPES = [(40,), (6, 40), (2, 3, 40), (2, 1, 3, 40), (0, 3, 40)]


def normal(*shape, seed=0, grad=True):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return torch.randn(*shape, generator=g).to(DEV).requires_grad_(grad)


def calls(shape, grad=True):
    def arg(*s, seed):
        return normal(*s, seed=seed, grad=grad)
    x = arg(*shape, seed=1)
    r = arg(*shape[:-1], 24, seed=2)
    g, h = arg(40, seed=3), arg(40, seed=4)
    w, b = arg(24, 40, seed=5), arg(24, seed=6)
    w2, b2 = arg(40, 24, seed=7), arg(40, seed=8)
    return {
        "norm": (gt.layer_norm, (x, g, h)),
        "norm8": (lambda *a: gt.layer_norm(*a, act8=True), (x, g, h)),
        "linear": (gt.linear_act, (x, w, b, r)),
        "gelu8": (lambda *a: gt.linear_act(*a, act="gelu", act8=True),
                  (x, w, b, r)),
        "block": (gt.ffn_block, (x, g, h, w, b, w2, b2)),
        "block8": (lambda *a: gt.ffn_block(*a, act8=True),
                   (x, g, h, w, b, w2, b2)),
    }


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("name", NAMES)
def test_in_place_after_a_call(shape, name):
    call, args = calls(shape)[name]

    def changed(in_place):
        y = call(*args)
        if in_place:
            y.mul_(3).add_(0.5)
            F.relu_(y)
        else:
            y = F.relu(y * 3 + 0.5)
        return [y.detach(), *torch.autograd.grad(y, args, y.detach())]
    for a, b in zip(changed(True), changed(False)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("name", NAMES)
def test_in_place_with_gradients_after_a_call_without(shape, name):
    call, args = calls(shape, grad=False)[name]
    with torch.no_grad():
        y = call(*args)
    for z in (y, call(*args)):
        assert not z._is_view() and z.is_contiguous()
        by = normal(z.shape[-1], seed=9)
        want = z * by
        z.mul_(by)
        assert torch.equal(z, want) and z.requires_grad


@pytest.mark.parametrize("shape", SHAPES)
def test_in_place_on_the_8_bit_form(shape):
    with torch.no_grad():
        p = gt.act8_pack(normal(*shape, grad=False))
        x = gt.act8_unpack(*p)
    assert not any(v._is_view() for v in (*p, x))
    x.mul_(normal(40, seed=9))
    p.scales.mul_(normal(1, seed=9))
    assert x.requires_grad and p.scales.requires_grad
