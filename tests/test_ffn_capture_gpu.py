"""Captured feed-forward calls under autocast: the parameters that are cast are
leaves of the captured graph, too."""
import pytest
import torch

import gtopkssgd_amd as gt

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def calls():
    torch.manual_seed(0)
    block = gt.FFNBlock(40, 72).to(DEV)
    linear = gt.FusedLinearAct(40, 24, act="gelu").to(DEV)
    x = torch.randn(30, 40, device=DEV, requires_grad=True)
    r = torch.randn(30, 24, device=DEV, requires_grad=True)
    half = torch.randn(24, dtype=torch.float16, device=DEV, requires_grad=True)
    w = linear.weight
    hooked = gt.FFNBlock(40, 72).to(DEV)
    hooked.fc2.register_forward_hook(lambda m, a, y: None)
    return {
        "hooked": (lambda: hooked(x), [x, *hooked.parameters()]),
        "block": (lambda: block(x), [x, *block.parameters()]),
        "linear": (lambda: linear(x, r), [x, r, *linear.parameters()]),
        "bias": (lambda: gt.linear_act(x, w, half), [x, w, half]),
    }


@pytest.mark.parametrize("name", ["block", "hooked", "linear", "bias"])
def test_a_living_graph_of_cast_leaves_is_refused(name):
    call, leaves = calls()[name]

    def step():
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = call()
        return torch.autograd.grad(y, leaves, torch.ones_like(y))
    want = step()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        living = call()
    graph = torch.cuda.CUDAGraph()
    mark = torch.zeros(1, device=DEV)
    with pytest.raises(RuntimeError, match="free that graph"):
        with torch.cuda.graph(graph):
            mark += 1
            with torch.autocast("cuda", dtype=torch.bfloat16):
                call()
    del living, graph
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        step()
