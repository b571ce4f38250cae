"""The block calls its children where something hangs on their being called."""
import copy

import pytest
import torch
from torch import nn
from torch.nn.modules import module as nn_module
from torch.nn.utils import parametrize, parametrizations, prune

import gtopkssgd_amd as gt

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]
CHILDREN = ["norm", "fc1", "fc2"]
# sums of up to 48 fp32 terms in another order, twice over
TOL = dict(rtol=0, atol=1e-4)


def block(device, **kwargs):
    torch.manual_seed(0)
    b = gt.FFNBlock(24, 48, **kwargs).to(device)
    with torch.no_grad():
        b.norm.weight.uniform_(0.5, 1.5)
        b.norm.bias.uniform_(-0.5, 0.5)
    x = torch.randn(2, 5, 24, generator=torch.Generator().manual_seed(1))
    return b, x.to(device).requires_grad_(True)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("child", CHILDREN)
@pytest.mark.parametrize("act", ["relu", "gelu"])
def test_forward_hooks_run(device, child, act):
    b, x = block(device, act=act)
    want = b(x)
    seen = []
    m = getattr(b, child)
    hooks = [m.register_forward_pre_hook(lambda m, a: seen.append(a[0].shape)),
             m.register_forward_hook(lambda m, a, y: seen.append(y.shape))]
    y = b(x)
    assert torch.allclose(y, want, **TOL)
    wide = {"norm": (24, 24), "fc1": (24, 48), "fc2": (48, 24)}[child]
    assert seen == [(2, 5, wide[0]), (2, 5, wide[1])]
    for h in hooks:
        h.remove()
    assert torch.equal(b(x), want)
    assert len(seen) == 2


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("child", CHILDREN)
def test_a_hook_that_changes_the_result_does(device, child):
    b, x = block(device)
    want = b(x)
    getattr(b, child).register_forward_hook(lambda m, a, y: y * 0)
    y = b(x)
    assert not torch.allclose(y, want, **TOL)
    if child == "fc2":
        assert torch.equal(y, x)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("child", CHILDREN)
def test_backward_hooks_run(device, child):
    b, x = block(device)
    want = torch.autograd.grad(b(x).sum(), [x, *b.parameters()])
    seen = []
    m = getattr(b, child)
    m.register_full_backward_pre_hook(lambda m, g: seen.append("before"))
    m.register_full_backward_hook(lambda m, i, o: seen.append("after"))
    got = torch.autograd.grad(b(x).sum(), [x, *b.parameters()])
    assert sorted(seen) == ["after", "before"]
    for p, q in zip(got, want):
        assert torch.allclose(p, q, rtol=1e-4, atol=1e-3)


@pytest.mark.parametrize("device", DEVICES)
def test_hooks_of_all_modules_run(device):
    b, x = block(device)
    seen = []
    handle = nn_module.register_module_forward_hook(
        lambda m, a, y: seen.append(m))
    try:
        b(x)
    finally:
        handle.remove()
    assert seen == [b.norm, b.fc1, b.fc2, b]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("act8", [False, True])
def test_pruned_weights_are_used_and_train(device, act8):
    b, x = block(device, act8=act8)
    prune.l1_unstructured(b.fc1, "weight", amount=0.5)
    b.eval()
    with torch.no_grad():
        one = b(x)
        b.fc1.weight_orig.mul_(2)
        two = b(x)
    assert not torch.allclose(one, two, **TOL)
    b.train()
    for _ in range(3):
        b.zero_grad()
        b(x).square().sum().backward()
        lost = b.fc1.weight_mask == 0
        assert (b.fc1.weight_orig.grad[lost] == 0).all()
        assert (b.fc1.weight_orig.grad[~lost] != 0).any()
    prune.remove(b.fc1, "weight")
    with torch.no_grad():
        assert torch.allclose(b(x), two, **TOL)


@pytest.mark.parametrize("device", DEVICES)
def test_parametrized_weights_are_used(device):
    b, x = block(device)
    parametrizations.weight_norm(b.fc2, "weight")
    one = b(x)
    with torch.no_grad():
        b.fc2.parametrizations.weight.original0.mul_(2)
    assert not torch.allclose(b(x), one, **TOL)
    b(x).sum().backward()
    assert b.fc2.parametrizations.weight.original0.grad is not None
    parametrize.remove_parametrizations(b.fc2, "weight")


class Low(nn.Module):
    """A layer and a product of low rank beside it."""

    def __init__(self, of, rank):
        super().__init__()
        self.of = of
        self.a = nn.Linear(of.in_features, rank, bias=False)
        self.b = nn.Linear(rank, of.out_features, bias=False)

    def forward(self, x):
        return self.of(x) + self.b(self.a(x))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("child", ["fc1", "fc2"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_children_put_in_their_place_are_called(device, child, act):
    b, x = block(device, act=act)
    want = b(x)
    low = Low(getattr(b, child), 3).to(device)
    setattr(b, child, low)
    y = b(x)
    assert not torch.allclose(y, want, **TOL)
    y.sum().backward()
    assert low.a.weight.grad is not None
    with torch.no_grad():
        low.b.weight.zero_()
    assert torch.allclose(b(x), want, **TOL)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("child", CHILDREN)
def test_layers_of_torchs_own_in_their_place(device, child):
    b, x = block(device)
    want = b(x)
    old = getattr(b, child)
    new = nn.LayerNorm(24) if child == "norm" else \
        nn.Linear(old.in_features, old.out_features)
    new.load_state_dict(old.state_dict())
    setattr(b, child, new.to(device))
    assert torch.allclose(b(x), want, **TOL)
    with torch.no_grad():
        new.weight.mul_(2)
    assert not torch.allclose(b(x), want, **TOL)
    b.norm = nn.Identity()
    b(x).sum().backward()


@pytest.mark.parametrize("device", DEVICES)
def test_an_activation_in_a_childs_place_is_applied(device):
    b, x = block(device, act="none")
    want = b(x)
    relu = gt.FusedLinearAct(24, 48, act="relu").to(device)
    relu.load_state_dict(b.fc1.state_dict())
    b.fc1 = relu
    assert not torch.allclose(b(x), want, **TOL)


@pytest.mark.gpu
@pytest.mark.parametrize("hooked", [False, True])
def test_types_under_autocast(hooked):
    b, x = block("cuda:0")
    if hooked:
        b.fc1.register_forward_hook(lambda m, a, y: None)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = b(x)
    assert y.dtype == torch.bfloat16
    y.float().sum().backward()
    assert all(p.grad.dtype == torch.float32 for p in [x, *b.parameters()])


@pytest.mark.parametrize("device", DEVICES)
def test_state_and_initial_values_are_as_before(device):
    """The children have the names and the first values of a layer norm and
    two linear layers that are made in this order."""
    torch.manual_seed(3)
    b = gt.FFNBlock(24, 48).to(device)
    torch.manual_seed(3)
    norm, fc1, fc2 = nn.LayerNorm(24), nn.Linear(24, 48), nn.Linear(48, 24)
    want = {f"{n}.{k}": v for n, m in (("norm", norm), ("fc1", fc1),
                                       ("fc2", fc2))
            for k, v in m.state_dict().items()}
    got = b.state_dict()
    assert list(got) == list(want)
    assert all(torch.equal(got[k].cpu(), want[k]) for k in want)
    c = copy.deepcopy(b)
    c.load_state_dict({k: v + 1 for k, v in want.items()})
    assert all(torch.equal(v.cpu(), want[k] + 1)
               for k, v in c.state_dict().items())
