"""The feed-forward operators' CPU form under forward mode: refused as well."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import gtopkssgd_amd as gt

X, G, W1, W2 = (torch.randn(*s) for s in ((5, 8), (8,), (16, 8), (8, 16)))


@pytest.mark.parametrize("call", [
    lambda x: gt.layer_norm(x, G), lambda x: gt.linear_act(x, W1, act="gelu"),
    lambda x: gt.ffn_block(x, G, None, W1, None, W2, None)])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(call, grad):
    with fwd.dual_level():
        x = fwd.make_dual(X.clone().requires_grad_(grad), torch.ones_like(X))
        with pytest.raises((RuntimeError, NotImplementedError)):
            call(x)


@pytest.mark.parametrize("call", [
    lambda x: gt.layer_norm(x, G), lambda x: gt.linear_act(x, W1, act="gelu")])
def test_traced_calls_compute(call):
    """Tracing sees the CPU form's own operations, or refuses it."""
    try:
        traced = torch.jit.trace(call, (X,), check_trace=False)
    except RuntimeError:
        return
    y = torch.randn(5, 8)
    assert torch.equal(traced(y), call(y))
