"""Feed-forward operators under what programs put round them: recomputed and
offloaded activations, inference mode, scaled losses, frozen parts."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

import gtopkssgd_amd as gt

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def parts(dtype=torch.bfloat16, act8=False):
    torch.manual_seed(0)
    block = gt.FFNBlock(40, 88, act8=act8).to(DEV, dtype)
    x = torch.randn(3, 11, 40, device=DEV).to(dtype).requires_grad_(True)
    return block, x, torch.randn(3, 11, 40, device=DEV).to(dtype)


@pytest.mark.parametrize("act8", [False, True])
@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_activations(act8, reentrant):
    block, x, dy = parts(act8=act8)
    leaves = [x, *block.parameters()]
    block(x).backward(dy)
    want = [p.grad.clone() for p in leaves]
    for p in leaves:
        p.grad = None
    checkpoint(block, x, use_reentrant=reentrant).backward(dy)
    assert all(torch.equal(p.grad, w) for p, w in zip(leaves, want))


@pytest.mark.parametrize("act8", [False, True])
def test_activations_kept_on_the_host(act8):
    block, x, dy = parts(act8=act8)
    leaves = [x, *block.parameters()]
    want = torch.autograd.grad(block(x), leaves, dy)
    with torch.autograd.graph.save_on_cpu():
        y = block(x)
    got = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_inference_mode():
    block, x, _ = parts()
    want = block(x)
    with torch.inference_mode():
        y = block(x)
        assert torch.equal(y, want) and not y.requires_grad
        assert torch.equal(block(y), block(want.detach()))


@pytest.mark.parametrize("frozen", ["norm", "fc1", "fc2", "norm fc1 fc2"])
def test_frozen_children(frozen):
    block, x, dy = parts()
    all_leaves = [x, *block.parameters()]
    every = torch.autograd.grad(block(x), all_leaves, dy)
    want = {id(p): g for p, g in zip(all_leaves, every)}
    for name in frozen.split():
        getattr(block, name).requires_grad_(False)
    leaves = [p for p in all_leaves if p.requires_grad]
    got = torch.autograd.grad(block(x), leaves, dy)
    for p, g in zip(leaves, got):
        assert torch.equal(g, want[id(p)])


def test_infinite_gradients_of_a_scaled_loss_show():
    """What a loss scaler looks for: an infinite dy leaves no finite gradient
    behind that it has a part in."""
    block, x, dy = parts(torch.float16)
    dy[1, 4, 7] = float("inf")
    got = torch.autograd.grad(block(x), [x, *block.parameters()], dy)
    assert all(not bool(torch.isfinite(g).all()) for g in got)
