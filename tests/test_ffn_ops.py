"""Feed-forward operators on the CPU: gradients against differences, the 8-bit
form by its definition, refusals, and the language model that uses them."""
import os
import subprocess
import sys

import pytest
import torch
from torch.autograd import gradcheck

import ffn_reference as ref
import gtopkssgd_amd as gt
from gtopkssgd_amd import models as zoo
from gtopkssgd_amd.trainer import DLTrainer

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ACTS = ["none", "relu", "gelu", "silu"]


def _double(*shape, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g, dtype=torch.double,
                       requires_grad=True)


@pytest.mark.parametrize("shape", [(5, 1), (1, 7), (2, 3, 9), (6,)])
@pytest.mark.parametrize("params", [True, False])
def test_norm_gradients_against_differences(shape, params):
    n = shape[-1]
    args = (_double(*shape, seed=1),) + (
        (_double(n, seed=2), _double(n, seed=3)) if params else ())
    assert gradcheck(lambda *a: gt.layer_norm(*a), args)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,res", [(True, True), (False, False)])
def test_linear_gradients_against_differences(act, bias, res):
    x, w = _double(2, 3, 7, seed=4), _double(5, 7, seed=5)
    b = _double(5, seed=6) if bias else None
    r = _double(2, 3, 5, seed=7) if res else None
    args = tuple(t for t in (x, w, b, r) if t is not None)

    def f(*a):
        a = list(a)
        x, w = a[:2]
        return gt.linear_act(x, w, a[2] if bias else None,
                             a[-1] if res else None, act=act)
    assert gradcheck(f, args)


@pytest.mark.parametrize("act", ["gelu", "relu"])
def test_block_gradients_against_differences(act):
    args = (_double(4, 6, seed=1), _double(6, seed=2), _double(6, seed=3),
            _double(10, 6, seed=4), _double(10, seed=5), _double(6, 10, seed=6),
            _double(6, seed=7))
    assert gradcheck(lambda *a: gt.ffn_block(*a, act=act), args)


def _edge_values():
    x = torch.randn(9, 300, generator=torch.Generator().manual_seed(0))
    x[0] = 0
    x[1, :128] *= 2.0 ** -140          # under the least scale
    x[2, 128:256] = 2.0 ** -119        # at it
    x[3, 5] = float("inf")
    x[4, 299] = float("nan")
    x[5, 200] = -float("inf")
    x[6] = torch.arange(300) - 150.0   # ties after scaling
    x[7, :128] = 254.0
    x[7, 1:128] = torch.arange(127) * 2.0 + 1.0
    x[8] = 3e38
    return x


def test_act8_by_its_definition():
    x = _edge_values()
    p = gt.act8_pack(x)
    assert p.codes.dtype == torch.int8 and p.codes.shape == x.shape
    assert p.scales.dtype == torch.float32 and p.scales.shape == (9, 3)
    back = gt.act8_unpack(*p)
    for r, c in ((3, 0), (4, 2), (5, 1)):
        lost = slice(128 * c, 128 * c + 128)
        assert torch.isnan(back[r, lost]).all()
        assert (p.codes[r, lost] == 0).all()
        rest = torch.ones(300, dtype=torch.bool)
        rest[lost] = False
        assert torch.isfinite(back[r, rest]).all()
    assert (back[0] == 0).all() and (back[1, :128] == 0).all()
    assert (p.codes[2, 128:256] == 127).all()
    fine = torch.tensor([0, 1, 2, 6, 7, 8])
    want = ref.pack_values(x[fine])
    assert torch.equal(back[fine], want.float())
    # half a code of the group's largest value, and the roundings of the two
    # factors and of the code's border
    a = torch.stack([x[fine][:, g:g + 128].abs().amax(1)
                     for g in (0, 128, 256)], 1).double()
    bound = (a / 127 * (0.5 + 127 * 4 * 2.0 ** -24)).repeat_interleave(
        128, 1)[:, :300] + 2.0 ** -119
    assert ((back[fine].double() - x[fine].double()).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16,
                                   torch.float32])
def test_act8_of_a_packed_value_is_itself(dtype):
    """Codes of values that are codes times a power of two come back whole."""
    g = torch.Generator().manual_seed(3)
    codes = torch.randint(-127, 128, (4, 200), generator=g)
    codes[:, 0] = 127
    codes[:, 128] = -127
    x = (codes * 0.25).to(dtype)
    p = gt.act8_pack(x)
    assert torch.equal(p.codes.long(), codes)


def test_act8_bound_on_gradients():
    """The gradient from 8 bits is the gradient of what they stand for."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(40, 300, generator=g)
    w = torch.randn(20, 300, generator=g, requires_grad=True)
    dy = torch.randn(40, 20, generator=g)
    gt.linear_act(x, w, act8=True).backward(dy)
    want, bound = ref.mm(dy.double().t(), ref.pack_values(x))
    ref.close(w.grad, want, bound + 2.0 ** -24 * want.abs())


def test_refusals_cpu():
    x, w, b = torch.randn(3, 8), torch.randn(5, 8), torch.randn(5)
    with pytest.raises(ValueError, match="unknown activation"):
        gt.linear_act(x, w, act="tanh")
    with pytest.raises(ValueError, match="unknown activation"):
        gt.FFNBlock(8, 16, act="tanh")
    with pytest.raises(RuntimeError, match="weight must have shape"):
        gt.linear_act(x, torch.randn(5, 7))
    with pytest.raises(RuntimeError, match="bias must have shape"):
        gt.linear_act(x, w, torch.randn(8))
    with pytest.raises(RuntimeError, match="residual must have"):
        gt.linear_act(x, w, b, residual=torch.randn(5))
    with pytest.raises(RuntimeError, match="weight must have shape"):
        gt.layer_norm(x, torch.randn(7))
    with pytest.raises(RuntimeError, match="last"):
        gt.layer_norm(torch.randn(3, 0))
    with pytest.raises(RuntimeError, match="last"):
        gt.act8_pack(torch.tensor(1.0))
    with pytest.raises(RuntimeError, match="scales must have shape"):
        gt.act8_unpack(torch.zeros(3, 200, dtype=torch.int8),
                       torch.zeros(3, 1))
    with pytest.raises(RuntimeError, match="int8"):
        gt.act8_unpack(torch.zeros(3, 200), torch.zeros(3, 2))
    with pytest.raises(RuntimeError, match="w2 must have shape"):
        gt.ffn_block(x, None, None, torch.randn(16, 8), None,
                     torch.randn(9, 16), None)
    with pytest.raises(ValueError, match="one dimension"):
        gt.FusedLayerNorm((3, 4))
    with pytest.raises(ValueError, match="ffn_mult"):
        zoo.lstm_ptb(50, 8, act8=True)
    x.requires_grad_(True)
    y = gt.layer_norm(x)
    dx, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_modules_share_state_with_torch():
    norm, plain = gt.FusedLayerNorm(12), torch.nn.LayerNorm(12)
    plain.load_state_dict(norm.state_dict())
    lin, lplain = gt.FusedLinearAct(12, 5, act="relu"), torch.nn.Linear(12, 5)
    lplain.load_state_dict(lin.state_dict())
    x = torch.randn(4, 12)
    # both round the same few operations, in another order
    assert torch.allclose(norm(x), plain(x), rtol=0, atol=64 * 2.0 ** -24)
    assert torch.allclose(lin(x), torch.relu(lplain(x)), rtol=0,
                          atol=64 * 2.0 ** -24 * 12)


def test_lstm_without_block_is_as_before():
    torch.manual_seed(0)
    a = zoo.lstm_ptb(60, 16)
    torch.manual_seed(0)
    b = zoo.create_net("lstm", "ptb", vocab_size=60, hidden=16)
    assert list(a.state_dict()) == list(b.state_dict())
    assert not any("ffn" in k for k in a.state_dict())
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q)


@pytest.mark.parametrize("act8", [False, True])
def test_lstm_with_block_trains(act8):
    tr = DLTrainer(dnn="lstm", dataset="ptb", batch_size=4, lr=0.1,
                   device="cpu", amp=False, num_workers=0, n_samples=64,
                   model_kwargs={"vocab_size": 120, "hidden": 24,
                                 "ffn_mult": 2, "act8": act8})
    opt = gt.DistributedOptimizer(
        tr.optimizer, tr.net.named_parameters(),
        compression=gt.compressors["gtopk"](0.05), density=0.05)
    before = tr.net.ffn.fc1.weight.detach().clone()
    for _ in range(2):
        loss = tr.train(1, dist_optimizer=opt)
        tr.update_model(dist_optimizer=opt)
    assert loss == loss
    assert not torch.equal(before, tr.net.ffn.fc1.weight)
    assert "perplexity" in tr.test()


def _train(*extra):
    return subprocess.run(
        [sys.executable, os.path.join(REPO, "train.py"), "--device", "cpu",
         "--no-amp", "--num-workers", "0", *extra],
        cwd=REPO, capture_output=True, text=True, timeout=300)


@pytest.mark.parametrize("extra", [
    ["--dnn", "mnistffn", "--ffn-mult", "2"],
    ["--dnn", "lstm", "--act8"],
    ["--dnn", "lstm", "--ffn-mult", "-1"]])
def test_train_command_refuses(extra):
    r = _train(*extra)
    assert r.returncode == 2 and "--ffn-mult" in r.stderr


def test_train_command_with_block(tmp_path):
    r = _train("--dnn", "lstm", "--dataset", "ptb", "--ffn-mult", "1",
               "--act8", "--batch-size", "2", "--max-epochs", "1",
               "--iters-per-epoch", "1", "--n-samples", "4",
               "--checkpoint-dir", str(tmp_path))
    assert r.returncode == 0, r.stderr[-2000:]
