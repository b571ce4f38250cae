"""What looks past an autograd function - forward mode, tracing, transforms of
functions - is refused by the feed-forward operators, never given a result
without its derivative or a graph without the kernel."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import gtopkssgd_amd as gt

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def normal(*shape, seed=0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return torch.randn(*shape, generator=g).to(torch.bfloat16).to(DEV)


# name, call, shapes of its arguments
CALLS = {
    "layer_norm": (gt.layer_norm, [(6, 40), (40,), (40,)]),
    "linear_act": (lambda x, w, b, r: gt.linear_act(x, w, b, r, act="gelu"),
                   [(6, 40), (24, 40), (24,), (6, 24)]),
    "ffn_block": (gt.ffn_block, [(6, 40), (40,), (40,), (24, 40), (24,),
                                 (40, 24), (40,)]),
}
EVERY = [(name, i) for name, (_, args) in CALLS.items()
         for i in range(len(args))]


def arguments(name):
    return [normal(*s, seed=i) for i, s in enumerate(CALLS[name][1])]


@pytest.mark.parametrize("name,i", EVERY)
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(name, i, grad):
    call, args = CALLS[name][0], arguments(name)
    with fwd.dual_level():
        args[i] = fwd.make_dual(args[i].requires_grad_(grad),
                                torch.ones_like(args[i]))
        with pytest.raises(RuntimeError, match="forward mode"):
            call(*args)


def test_forward_mode_of_the_8_bit_form_is_refused():
    codes = torch.ones(2, 5, dtype=torch.int8, device=DEV)
    scales = torch.ones(2, 1, device=DEV)
    with fwd.dual_level():
        dual = fwd.make_dual(scales, torch.ones_like(scales))
        with pytest.raises(RuntimeError, match="forward mode"):
            gt.act8_unpack(codes, dual)
        with pytest.raises(RuntimeError, match="forward mode"):
            gt.act8_pack(dual)
    with pytest.raises(RuntimeError, match="no gradient"):
        gt.act8_unpack(codes, scales.requires_grad_(True))
    with torch.no_grad():
        assert (gt.act8_unpack(codes, scales) == 1).all()


@pytest.mark.parametrize("name", list(CALLS) + ["act8"])
@pytest.mark.parametrize("grad", [False, True])
def test_tracing_is_refused(name, grad):
    if name == "act8":
        call, args = (lambda x: gt.act8_unpack(*gt.act8_pack(x))), [normal(6, 40)]
    else:
        call, args = CALLS[name][0], arguments(name)
    args = tuple(a.requires_grad_(grad) for a in args)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(call, args, check_trace=False)
    call(*args)


@pytest.mark.parametrize("name", list(CALLS))
def test_function_transforms_are_refused(name):
    call, args = CALLS[name][0], arguments(name)

    def of_x(x):
        return call(x, *args[1:])
    x3 = torch.stack([args[0], args[0]])
    with pytest.raises(RuntimeError, match="torch.func"):
        torch.vmap(of_x)(x3)
    with pytest.raises(RuntimeError, match="torch.func"):
        torch.func.grad(lambda x: of_x(x).float().sum())(args[0])
    with pytest.raises(RuntimeError, match="torch.func"):
        torch.func.jvp(of_x, (args[0],), (args[0],))


@pytest.mark.parametrize("name", list(CALLS))
@pytest.mark.parametrize("mode", ["real", "fake"])
def test_graphs_of_calls_are_refused(name, mode):
    from torch.fx.experimental.proxy_tensor import make_fx
    call, args = CALLS[name][0], arguments(name)
    with pytest.raises(RuntimeError):
        make_fx(call, tracing_mode=mode)(*args)


@pytest.mark.parametrize("name", list(CALLS))
def test_compiled_programs_call_them(name):
    """torch.compile leaves its graph for the call and goes on after it."""
    call = CALLS[name][0]
    args = [a.requires_grad_(True) for a in arguments(name)]

    def program(*a):
        return call(a[0] * 2, *a[1:]) + 1
    y = torch.compile(program, backend="eager")(*args)
    assert torch.equal(y, program(*args))
    got = torch.autograd.grad(y, args, torch.ones_like(y))
    want = torch.autograd.grad(program(*args), args, torch.ones_like(y))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
