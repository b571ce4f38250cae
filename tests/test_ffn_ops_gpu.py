"""Feed-forward operators on the MI355X against 64 bits on the CPU, value by
value, within the bounds of tests/ffn_reference.py."""
import pytest
import torch

import ffn_reference as ref
import gtopkssgd_amd as gt
from gtopkssgd_amd import models as zoo
from gtopkssgd_amd.trainer import DLTrainer

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
ACTS = ["none", "relu", "gelu", "silu"]


def make(*shape, t=FP, scale=1.0, shift=0.0, seed=0, grad=True):
    g = torch.Generator().manual_seed(seed + 1000 * len(shape) + sum(shape))
    v = torch.randn(*shape, generator=g) * scale + shift
    return v.to(t).to(DEV).requires_grad_(grad)


# ---- layer norm ---------------------------------------------------------------

def check_norm(x, w, b, dy, act8, eps=1e-5):
    t = x.dtype
    y = gt.layer_norm(x, w, b, eps, act8=act8)
    assert y.dtype == t and y.shape == x.shape
    leaves = [v for v in (x, w, b) if v is not None and v.requires_grad]
    grads = dict(zip([id(v) for v in leaves],
                     torch.autograd.grad(y, leaves, dy)))
    n = x.shape[-1]
    x2, d2 = ref.wide(x).reshape(-1, n), ref.wide(dy).reshape(-1, n)
    want = ref.norm(x2, ref.wide(w), ref.wide(b), eps, t, act8, d2,
                    ref.pack_values(x2) if act8 else None)
    ref.close(y, *want[0], what="y")
    if id(x) in grads:
        ref.close(grads[id(x)], *ref.rounded(*want[1], t), what="dx")
    for p, k in ((w, 2), (b, 3)):
        if p is not None and p.requires_grad:
            assert grads[id(p)].dtype == p.dtype
            ref.close(grads[id(p)], *ref.rounded(*want[k], p.dtype),
                      what=f"param {k}")


@pytest.mark.parametrize("dim", [1, 2, 3, 7, 8, 64, 127, 128, 129, 512, 1023,
                                 1500, 1501, 2048, 2049, 4097, 8193])
@pytest.mark.parametrize("t", [BF, HF, FP])
@pytest.mark.parametrize("act8", [False, True])
def test_norm_dims(dim, t, act8):
    # under 8 values a row's variance may vanish: eps is of the row's own size
    eps = 1e-5 if dim > 7 else 0.5
    check_norm(make(37, dim, t=t, scale=1.5, shift=0.25),
               make(dim, t=FP, scale=0.2, shift=1.0, seed=1),
               make(dim, t=FP, seed=2), make(37, dim, t=t, seed=3, grad=False),
               act8, eps)


@pytest.mark.parametrize("dim", [16384, 32768, 32769, 70001])
@pytest.mark.parametrize("act8", [False, True])
def test_norm_long_rows(dim, act8):
    check_norm(make(3, dim, t=BF), make(dim, t=BF, seed=1), make(dim, t=BF,
               seed=2), make(3, dim, t=BF, seed=3, grad=False), act8)


@pytest.mark.parametrize("rows", [1, 2, 4, 5, 3071, 4099])
@pytest.mark.parametrize("t", [BF, FP])
def test_norm_rows(rows, t):
    check_norm(make(rows, 200, t=t), make(200, t=t, seed=1),
               make(200, t=t, seed=2), make(rows, 200, t=t, seed=3,
                                            grad=False), False)


@pytest.mark.parametrize("which", ["x", "w", "b", "wb", "none"])
def test_norm_some_gradients(which):
    x = make(20, 130, t=BF, grad="x" in which or which == "none")
    w = None if which == "none" else make(130, seed=1, grad="w" in which)
    b = None if which == "none" else make(130, seed=2, grad="b" in which)
    check_norm(x, w, b, make(20, 130, t=BF, seed=3, grad=False), False)


def test_norm_strides():
    big = make(6, 50, 400, t=BF, grad=False)
    w, b = make(131, seed=1), make(131, seed=2)
    for x in (big[:, :, 1:132], big[::2, ::3, 7:138],
              big[:, :, :131].transpose(0, 1),
              big.permute(2, 0, 1)[:131].permute(1, 2, 0)):
        x = x.detach().requires_grad_(True)
        dy = torch.randn(1, 1, 131, generator=torch.Generator().manual_seed(
            1)).to(BF).to(DEV).expand(x.shape)
        check_norm(x, w, b, dy, True)
    wide = make(262, seed=5, grad=False)
    check_norm(make(9, 131, t=BF), wide[::2].detach().requires_grad_(True),
               wide[1::2].detach().requires_grad_(True),
               make(9, 131, t=BF, seed=6, grad=False), False)


def test_norm_no_rows_and_one_dimension():
    x, w = make(0, 40, t=BF), make(40, seed=1)
    y = gt.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert dx.shape == (0, 40) and (dw == 0).all()
    v = make(40, t=FP)
    check_norm(v, make(40, seed=1), make(40, seed=2),
               make(40, seed=3, grad=False), False)


@pytest.mark.parametrize("act8", [False, True])
def test_norm_bad_row_stays_in_its_row(act8):
    x = make(9, 300, t=BF, grad=False)
    x[2, 7], x[5, 299] = float("nan"), float("inf")
    x.requires_grad_(True)
    y = gt.layer_norm(x, act8=act8)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    bad = torch.tensor([2, 5], device=DEV)
    fine = torch.tensor([0, 1, 3, 4, 6, 7, 8], device=DEV)
    for v in (y, dx):
        assert torch.isnan(v[bad]).any(1).all()
        assert torch.isfinite(v[fine]).all()


def test_norm_equal_values():
    """A row of one value: nothing but the bias is left of it."""
    x = torch.full((3, 1000), 3.0, device=DEV, requires_grad=True)
    b = make(1000, seed=2)
    y = gt.layer_norm(x, None, b)
    assert torch.equal(y, b.expand(3, -1))


# ---- linear layer ---------------------------------------------------------------

def check_linear(x, w, b, res, act, act8, dy):
    t = x.dtype
    y = gt.linear_act(x, w, b, res, act=act, act8=act8)
    assert y.dtype == t and y.shape == (*x.shape[:-1], w.shape[0])
    leaves = [v for v in (x, w, b, res) if v is not None and v.requires_grad]
    grads = dict(zip([id(v) for v in leaves],
                     torch.autograd.grad(y, leaves, dy)))
    k, n = x.shape[-1], w.shape[0]
    want = ref.linear(ref.wide(x).reshape(-1, k), ref.wide(w), ref.wide(b),
                      None if res is None else ref.wide(res).reshape(-1, n),
                      act, t, act8, ref.wide(dy).reshape(-1, n))
    ref.close(y, *want[0], what="y")
    if id(x) in grads:
        ref.close(grads[id(x)], *want[1], what="dx")
    if id(w) in grads:
        ref.close(grads[id(w)], *want[2], what="dw")
    if b is not None and id(b) in grads:
        assert grads[id(b)].dtype == b.dtype
        ref.close(grads[id(b)], *ref.rounded(*want[3], b.dtype), what="db")
    if res is not None and id(res) in grads:
        assert torch.equal(grads[id(res)], dy)


def linear_case(m, k, n, t, act="none", res=False, act8=False, bias="t"):
    check_linear(
        make(m, k, t=t), make(n, k, t=t, scale=k ** -0.5, seed=1),
        None if bias is None else make(n, t=FP if bias == "fp32" else t,
                                       seed=2),
        make(m, n, t=t, seed=3) if res else None, act, act8,
        make(m, n, t=t, seed=4, grad=False))


@pytest.mark.parametrize("m,k,n", [
    (1, 1, 1), (1, 8, 1), (1, 1500, 70), (2, 3, 5), (3, 64, 64), (7, 63, 65),
    (16, 129, 127), (20, 1500, 300), (31, 100, 9), (33, 77, 257),
    (64, 128, 128), (65, 130, 67), (130, 257, 77), (257, 1501, 255),
    (300, 200, 301), (513, 40, 1), (700, 65, 520)])
@pytest.mark.parametrize("t", [BF, HF, FP])
def test_linear_sizes(m, k, n, t):
    linear_case(m, k, n, t, act="relu", res=True)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("t", [BF, HF, FP])
@pytest.mark.parametrize("res", [False, True])
@pytest.mark.parametrize("m,k,n", [(150, 140, 260), (9, 30, 41)])
def test_linear_acts(act, t, res, m, k, n):
    linear_case(m, k, n, t, act=act, res=res)


@pytest.mark.parametrize("bias", [None, "fp32"])
def test_linear_bias(bias):
    linear_case(50, 70, 90, BF, act="gelu", bias=bias)


@pytest.mark.parametrize("k", [1, 7, 63, 64, 128, 220, 255, 256, 300])
@pytest.mark.parametrize("m,n", [(1, 9), (70, 260), (2500, 40)])
@pytest.mark.parametrize("t,bias", [(BF, "t"), (HF, "fp32"), (FP, "t")])
def test_linear_bias_gradient_beside_the_weights(k, m, n, t, bias):
    """The last tile of dW has room for the sum of the rows, or has none; the
    sum over many rows goes in parts or in one."""
    linear_case(m, k, n, t, bias=bias)


def on_lines(v):
    ld = -(-v.shape[1] // 64) * 64
    out = torch.full((v.shape[0], ld), float("nan"), dtype=v.dtype, device=DEV)
    out = out[:, :v.shape[1]]
    out.copy_(v.detach())
    return out.requires_grad_(v.requires_grad)


@pytest.mark.parametrize("t", [BF, HF])
@pytest.mark.parametrize("act,act8", [("none", False), ("gelu", True)])
def test_linear_copies_long_operands(t, act, act8):
    """Operands that are copied to rows on lines: the same bits as from operands
    that lie so, and some rows against 64 bits."""
    m, k, n = 20000, 499, 20100
    x, w = make(m, k, t=t), make(n, k, t=t, scale=k ** -0.5, seed=1)
    b = make(n, t=t, seed=2)
    dy = make(m, n, t=t, seed=3, grad=False)
    got = gt.linear_act(x, w, b, act=act, act8=act8)
    lines = [on_lines(x), on_lines(w), b]
    want = gt.linear_act(*lines, act=act, act8=act8)
    assert torch.equal(got, want)
    with torch.no_grad():
        assert torch.equal(gt.linear_act(x, w, b, act=act), want)
    rows = [0, 1, 777, m - 1]
    sample = ref.linear(ref.wide(x[rows]), ref.wide(w), ref.wide(b), None, act,
                        t, act8, ref.wide(dy[rows]))
    ref.close(got[rows], *sample[0], what="y")
    got = torch.autograd.grad(got, [x, w, b], dy)
    want = torch.autograd.grad(want, lines, dy)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    ref.close(got[0][rows], *sample[1], what="dx")


@pytest.mark.parametrize("m,k,n", [(8000, 2570, 2900), (20001, 1500, 2000),
                                   (30000, 1023, 777), (12345, 256, 4100),
                                   (9000, 3900, 3900)])
@pytest.mark.parametrize("t", [BF, HF])
def test_linear_long_weight_gradients(m, k, n, t):
    """Sums over many rows, whole and in parts, against 64 bits: half a step of
    rounding, and the rounding of m additions in fp32."""
    x = make(m, k, t=t, grad=False)
    w, b = make(n, k, t=t, seed=1), make(n, t=t, seed=2)
    dy = make(m, n, t=t, seed=3, grad=False)
    dw, db = torch.autograd.grad(gt.linear_act(x, w, b), [w, b], dy)
    xd, d = x.double(), dy.double().t().contiguous()
    for got, one in ((dw, xd), (db[:, None], torch.ones_like(xd[:, :1]))):
        want = torch.mm(d, one)
        bound = want.abs() * torch.finfo(t).eps / 2 + \
            torch.mm(d.abs(), one.abs()) * m * 2.0 ** -24 + 2.0 ** -24
        assert bool(((got.double() - want).abs() <= bound).all())
    again = torch.autograd.grad(gt.linear_act(x, w, b), [w, b], dy)
    assert torch.equal(again[0], dw) and torch.equal(again[1], db)


def test_block_copies_long_weights():
    args = block_args(20000, 499, 9001, BF)
    dy = make(20000, 499, t=BF, seed=9, grad=False)
    lines = list(args)
    lines[3], lines[5] = on_lines(args[3]), on_lines(args[5])
    ys = [gt.ffn_block(*a, act8=True) for a in (args, lines)]
    assert torch.equal(*ys)
    with torch.no_grad():
        assert torch.equal(gt.ffn_block(*args), ys[0])
    got, want = (torch.autograd.grad(y, a, dy) for y, a in zip(ys, (args, lines)))
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("m,k,n", [(2500, 300, 40), (40, 3100, 70),
                                   (70, 50, 2500), (2100, 520, 530)])
@pytest.mark.parametrize("t", [BF, FP])
def test_linear_long_sums(m, k, n, t):
    """Few tiles and long sums: the product is split and joined."""
    linear_case(m, k, n, t, act="relu", res=True)


@pytest.mark.parametrize("act", ["none", "relu"])
@pytest.mark.parametrize("t", [BF, HF, FP])
@pytest.mark.parametrize("m,k,n", [(150, 140, 260), (9, 129, 41), (1, 1, 1)])
def test_linear_act8(act, t, m, k, n):
    linear_case(m, k, n, t, act=act, res=True, act8=True)


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("t", [BF, HF, FP])
@pytest.mark.parametrize("m,k,n", [(150, 140, 260), (9, 30, 41), (300, 64, 128)])
def test_linear_act8_smooth(act, t, m, k, n):
    """x and W are small integers over a power of two, so that u is exact in
    every order of summing and its codes are the reference's."""
    g = torch.Generator().manual_seed(m)
    x = (torch.randint(-4, 5, (m, k), generator=g) / 4).to(t).to(DEV)
    w = (torch.randint(-4, 5, (n, k), generator=g) / 8).to(t).to(DEV)
    b = (torch.randint(-4, 5, (n,), generator=g) / 8).to(t).to(DEV)
    check_linear(x.requires_grad_(True), w.requires_grad_(True),
                 b.requires_grad_(True), make(m, n, t=t, seed=3), act, True,
                 make(m, n, t=t, seed=4, grad=False))


@pytest.mark.parametrize("t", [BF, FP])
def test_linear_strides(t):
    big = make(5, 60, 400, t=t, grad=False)
    wbig = make(220, 300, t=t, scale=0.1, seed=1, grad=False)
    for x, w in ((big[:, :, 1:132], wbig[:77, 3:134]),
                 (big[::2, ::3, 2:133], wbig[::2, :131]),
                 (big[:, :, :220].transpose(0, 1), wbig[:, :131].t()[:, :220]),
                 (big.permute(2, 0, 1)[:131].permute(1, 2, 0),
                  wbig[1:, 1:132])):
        x = x.detach().requires_grad_(True)
        w = w.detach().requires_grad_(True)
        n = w.shape[0]
        res = make(*x.shape[:-1], n + 3, t=t, seed=2, grad=False)[..., 1:n + 1]
        dy = make(1, 1, n, t=t, seed=3, grad=False).expand(*x.shape[:-1], n)
        check_linear(x, w, None, res.detach().requires_grad_(True), "relu",
                     False, dy)


@pytest.mark.parametrize("which", ["x", "w", "b", "r", "xw"])
def test_linear_some_gradients(which):
    check_linear(make(40, 50, t=BF, grad="x" in which),
                 make(60, 50, t=BF, seed=1, scale=0.1, grad="w" in which),
                 make(60, t=BF, seed=2, grad="b" in which),
                 make(40, 60, t=BF, seed=3, grad="r" in which), "gelu", False,
                 make(40, 60, t=BF, seed=4, grad=False))


def test_linear_no_rows():
    x, w, b = make(0, 40, t=BF), make(30, 40, t=BF, seed=1), make(30, t=BF)
    for act in ACTS:
        y = gt.linear_act(x, w, b, act=act, act8=act == "gelu")
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
        assert dx.shape == (0, 40) and (dw == 0).all() and (db == 0).all()


@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("k", [77, 128, 1501])
def test_linear_bad_values_stay_in_their_row(m, k):
    """What lies behind a row's last value, infinities and NaN among it, does
    not reach it; a bad row of x reaches only its own."""
    store = torch.full((m + 1, k + 3), float("nan"), device=DEV, dtype=BF)
    x = store[:m, 1:k + 1]
    x.copy_(make(m, k, t=BF, grad=False))
    wstore = torch.full((71, k + 3), float("inf"), device=DEV, dtype=BF)
    w = wstore[:70, 2:k + 2]
    w.copy_(make(70, k, t=BF, seed=1, scale=0.1, grad=False))
    check_linear(x.detach().requires_grad_(True),
                 w.detach().requires_grad_(True), None, None, "none", False,
                 make(m, 70, t=BF, seed=2, grad=False))
    if m > 1:
        bad = x.clone()
        bad[m // 2, k - 1] = float("nan")
        y = gt.linear_act(bad, w)
        rows = torch.isnan(y).any(1).nonzero().flatten().tolist()
        assert rows == [m // 2]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("t", [BF, HF, FP])
@pytest.mark.parametrize("m", [5, 70])
def test_linear_infinite_values(act, t, m):
    """Where u is infinite, every activation of it is, and its slope is 1; it
    is NaN where u is."""
    k, n = 40, 24
    x = make(m, k, t=t)
    w = make(n, k, t=t, seed=1)
    with torch.no_grad():
        x[1, 3] = float("inf")
        x[3, 3] = float("nan")
        w[:, 3] = w[:, 3].abs() + 0.125
    dy = make(m, n, t=t, seed=2, grad=False)
    y = gt.linear_act(x, w, act=act)
    assert bool((y[1] == float("inf")).all())
    assert bool(torch.isnan(y[3]).all())
    dx, = torch.autograd.grad(y, x, dy)
    straight, = torch.autograd.grad(gt.linear_act(x, w), x, dy)
    assert torch.equal(dx[1], straight[1])
    if act in ("gelu", "silu"):
        assert bool(torch.isnan(dx[3]).all())
    others = [i for i in range(m) if i not in (1, 3)]
    assert bool(torch.isfinite(y[others]).all() & torch.isfinite(dx[others]).all())


def test_linear_keeps_results_without_gradients():
    x, w = make(33, 77, t=BF), make(50, 77, t=BF, seed=1)
    y = gt.linear_act(x, w, act="gelu")
    with torch.no_grad():
        assert torch.equal(y, gt.linear_act(x, w, act="gelu"))


def test_far_offsets():
    """Rows whose place needs more than 32 bits, in values and in bytes."""
    rows, k = 300_000, 8192
    x = torch.zeros(rows, k, device=DEV, dtype=BF)
    part = make(3, k, t=BF, grad=False)
    at = torch.tensor([0, 262_145, rows - 1], device=DEV)
    x[at] = part
    w = make(8, k, t=BF, scale=0.01, seed=1, grad=False)
    assert torch.equal(gt.linear_act(x, w)[at], gt.linear_act(part, w)) or \
        torch.allclose(gt.linear_act(x, w)[at].float(),
                       gt.linear_act(part, w).float(), rtol=2.0 ** -7,
                       atol=1e-4)
    y = gt.layer_norm(x)
    assert torch.equal(y[at], gt.layer_norm(part))
    assert (y[1] == 0).all() and (y[rows - 2] == 0).all()
    del y
    p = gt.act8_pack(x)
    q = gt.act8_pack(part)
    assert torch.equal(p.codes[at], q.codes)
    assert torch.equal(p.scales[at], q.scales)
    del p
    # across k: dW sums over all rows; only three of them are not zero
    xs, ws = x.requires_grad_(True), w.clone().requires_grad_(True)
    dy = torch.zeros(rows, 8, device=DEV, dtype=BF)
    dy[at] = make(3, 8, t=BF, seed=5, grad=False)
    dw, = torch.autograd.grad(gt.linear_act(xs, ws), ws, dy)
    want, bound = ref.mm(ref.wide(dy[at]).t(), ref.wide(part))
    ref.close(dw, *ref.rounded(want, bound, BF))


# ---- 8-bit form -----------------------------------------------------------------

@pytest.mark.parametrize("t", [BF, HF, FP])
@pytest.mark.parametrize("shape", [(1,), (1, 1), (5, 7), (33, 1501), (2, 3, 128),
                                   (4, 129), (700, 256), (0, 9), (3, 6000)])
def test_act8_is_the_cpu_one(t, shape):
    x = torch.randn(*shape, generator=torch.Generator().manual_seed(1))
    if x.dim() > 1:
        x = x * torch.exp2(torch.randn(*shape[:-1], 1) * 3)
    x = x.to(t)
    p, q = gt.act8_pack(x.to(DEV)), gt.act8_pack(x)
    assert torch.equal(p.codes.cpu(), q.codes)
    assert torch.equal(p.scales.cpu(), q.scales)
    for o in (BF, HF, FP):
        assert torch.equal(gt.act8_unpack(*p, o).cpu(),
                           gt.act8_unpack(*q, o))


def test_act8_edges_are_the_cpu_ones():
    from test_ffn_ops import _edge_values
    x = _edge_values()
    p, q = gt.act8_pack(x.to(DEV)), gt.act8_pack(x)
    assert torch.equal(p.codes.cpu(), q.codes)
    assert torch.equal(p.scales.cpu().nan_to_num(-1), q.scales.nan_to_num(-1))


@pytest.mark.parametrize("shape", [(5, 200), (3, 2, 200), (200,)])
def test_act8_pack_of_a_leaf_is_not_differentiable(shape):
    x = make(*shape).transpose(0, -1) if len(shape) > 2 else make(*shape)
    p = gt.act8_pack(x)
    assert not p.codes.requires_grad and not p.scales.requires_grad
    assert p.scales.grad_fn is None
    back = gt.act8_unpack(*p)
    assert back.shape == x.shape and not back.requires_grad


def test_act8_more_chunks_than_threads():
    """9 rows of 2^30 - 8 values: more chunks of 8 than one launch has threads
    for, the last of them against the codes."""
    rows, dim = 9, 2 ** 30 - 8
    codes = torch.zeros(rows, dim, dtype=torch.int8, device=DEV)
    codes[-1, -1000:] = torch.arange(1000, device=DEV).sub(500).clamp(-127, 127)
    codes[0, :3] = 7
    scales = torch.full((rows, -(-dim // 128)), 0.5, device=DEV)
    x = gt.act8_unpack(codes, scales, BF)
    assert torch.equal(x[-1, -1000:], codes[-1, -1000:].to(BF) * 0.5)
    assert torch.equal(x[0, :8], codes[0, :8].to(BF) * 0.5)
    assert not bool(x[-2].any())


def test_act8_strides():
    x = make(40, 300, t=BF, grad=False)
    for v in (x[:, 1:132], x[::3, :131], x.t()):
        p, q = gt.act8_pack(v), gt.act8_pack(v.contiguous().cpu())
        assert torch.equal(p.codes.cpu(), q.codes)
        assert torch.equal(p.scales.cpu(), q.scales)


# ---- the block ---------------------------------------------------------------------

NAMES = ["x", "norm_weight", "norm_bias", "w1", "b1", "w2", "b2"]


def block_args(rows, d, h, t, pt=None, grad=True):
    pt = pt or t
    return [make(rows, d, t=t, grad=grad),
            make(d, t=pt, scale=0.2, shift=1.0, seed=1, grad=grad),
            make(d, t=pt, scale=0.2, seed=2, grad=grad),
            make(h, d, t=t, scale=d ** -0.5, seed=3, grad=grad),
            make(h, t=pt, scale=0.1, seed=4, grad=grad),
            make(d, h, t=t, scale=h ** -0.5, seed=5, grad=grad),
            make(d, t=pt, scale=0.1, seed=6, grad=grad)]


def composed(x, nw, nb, w1, b1, w2, b2, act, act8):
    h = gt.layer_norm(x, nw, nb, act8=act8)
    a = gt.linear_act(h, w1, b1, act=act, act8=act8)
    return gt.linear_act(a, w2, b2, residual=x, act8=act8)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("act8", [False, True])
@pytest.mark.parametrize("t", [BF, HF, FP])
@pytest.mark.parametrize("rows,d,h", [(1, 16, 64), (37, 100, 401),
                                      (300, 128, 512), (515, 65, 130)])
def test_block_is_its_operators(act, act8, t, rows, d, h):
    """The block may take other tiles than the operators by themselves, and so
    add in another order: sums of n terms are off by (n + 8) 2^-24 times the
    terms' sizes, which are sqrt(n) of the sum's own where signs vary; then a
    value may round the other way, by two half steps, and so may what it is
    made from.  The gradients also differ by where p and dx round."""
    args = block_args(rows, d, h, t)
    dy = make(rows, d, t=t, seed=9, grad=False)
    y = gt.ffn_block(*args, act=act, act8=act8)
    z = composed(*args, act, act8)
    n = max(d, h)
    far = 2 * (n + 8) * ref.E * n ** 0.5
    limit = 6 * ref.U[t] + far
    assert (y - z).double().norm() <= limit * z.double().norm()
    got = torch.autograd.grad(y, args, dy)
    want = torch.autograd.grad(z, args, dy)
    for n, a, b in zip(NAMES, got, want):
        a, b = a.double(), b.double()
        # six roundings at most lie between the two, each U of the size of a
        # tensor that the result is a sum over: in the 2-norm they add up as
        # if all went one way
        limit = max(6 * ref.U[t] * 2, 2e-6)
        if act8:
            # A value that is off by `far` of its size, a code's step being
            # a / 127 of the group's largest a, takes another code with a
            # chance of 127 far at most, and is then off by a step.  a is under
            # 4 times a group's own size for normal values: in the 2-norm 4 /
            # 127 times the root of the share.
            limit += (127 * far) ** 0.5 * 4 / 127
        assert (a - b).norm() <= limit * b.norm() + 1e-6, n


@pytest.mark.parametrize("act,t", [("gelu", BF), ("silu", HF), ("gelu", FP),
                                   ("relu", BF)])
def test_block_against_64_bits(act, t):
    rows, d, h = 220, 96, 384
    args = block_args(rows, d, h, t)
    dy = make(rows, d, t=t, seed=9, grad=False)
    got = torch.autograd.grad(gt.ffn_block(*args, act=act), args, dy)
    wide = [ref.wide(a).requires_grad_(True) for a in args]
    y = gt.ffn_block(*wide, act=act)          # the CPU's, in 64 bits
    want = torch.autograd.grad(y, wide, ref.wide(dy))
    ref_y = gt.ffn_block(*args, act=act).double().cpu()
    # h, a, da, p, dh and the result round: at most six times U in the 2-norm,
    # and 2e-6 for fp32's sums of up to 384 terms (384 * 2^-24 at worst)
    limit = 6 * ref.U[t] + 384 * ref.E
    if act == "relu":
        # Where u is within its error of 0 the slope jumps.  The error is at
        # most U of u's deviation s in the 2-norm, and u's density at 0 is
        # 0.4 / s: a share of 2 * 0.4 U of the values, twice that of the half
        # that relu lets through, in the 2-norm its root.
        limit += (1.6 * ref.U[t]) ** 0.5
    assert (ref_y - y.detach()).norm() <= limit * y.detach().norm()
    for n, a, b in zip(NAMES, got, want):
        assert (a.double().cpu() - b).norm() <= limit * b.norm(), n


def test_block_gradient_against_differences():
    """fp32 gradients along a direction, against central differences in 64
    bits; h = 1e-4 leaves h^2 / 6 of the third derivative, some 1e-8."""
    args = block_args(40, 48, 96, FP)
    dy = make(40, 48, seed=9, grad=False)
    got = torch.autograd.grad(gt.ffn_block(*args), args, dy)
    wide = [ref.wide(a) for a in args]
    for i, n in enumerate(NAMES):
        g = torch.Generator().manual_seed(i)
        v = torch.randn(wide[i].shape, generator=g, dtype=torch.double)

        def f(s):
            a = list(wide)
            a[i] = a[i] + s * v
            return (gt.ffn_block(*a) * ref.wide(dy)).sum()
        want = (f(1e-4) - f(-1e-4)) / 2e-4
        have = (got[i].double().cpu() * v).sum()
        # 96 + 48 + 40 terms deep in fp32, in the 2-norm
        limit = 184 * ref.E * got[i].double().norm().cpu() * v.norm() + 1e-6
        assert (have - want).abs() <= limit, n


def test_block_without_parameters_that_may_lack():
    args = block_args(30, 40, 80, BF)
    y = gt.ffn_block(args[0], None, None, args[3], None, args[5], None)
    z = composed(args[0], None, None, args[3], None, args[5], None, "gelu",
                 False)
    assert (y - z).float().norm() <= 6 * ref.U[BF] * z.float().norm()
    got = torch.autograd.grad(y, [args[0], args[3], args[5]],
                              torch.ones_like(y))
    assert all(torch.isfinite(g).all() for g in got)


@pytest.mark.parametrize("which", range(7))
def test_block_one_gradient(which):
    args = block_args(50, 40, 90, BF)
    dy = make(50, 40, t=BF, seed=9, grad=False)
    every = torch.autograd.grad(gt.ffn_block(*args, act8=True), args, dy)
    some = [a.detach().requires_grad_(i == which) for i, a in enumerate(args)]
    one, = torch.autograd.grad(gt.ffn_block(*some, act8=True), [some[which]],
                               dy)
    limit = 4 * ref.U[BF]  # p may be kept in one part or two
    assert (one - every[which]).double().norm() <= \
        limit * every[which].double().norm()


def test_block_no_rows():
    args = block_args(0, 40, 80, BF)
    y = gt.ffn_block(*args, act8=True)
    got = torch.autograd.grad(y, args, torch.empty_like(y))
    assert got[0].shape == (0, 40)
    assert all((g == 0).all() for g in got[1:])


# ---- as programs use them ------------------------------------------------------------

@pytest.mark.parametrize("act8", [False, True])
@pytest.mark.parametrize("t,rows,d,h", [(BF, 700, 300, 1200), (FP, 64, 40, 100),
                                        (BF, 2000, 64, 64)])
def test_same_bits_each_time(act8, t, rows, d, h):
    args = block_args(rows, d, h, t)
    dy = make(rows, d, t=t, seed=9, grad=False)

    def once():
        y = gt.ffn_block(*args, act8=act8)
        return [y, *torch.autograd.grad(y, args, dy)]
    a, b = once(), once()
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("rows", [5, 90])
def test_one_tensor_twice(rows):
    """x as its own residual and weight: both edges get their gradients."""
    v = make(rows, rows, t=FP, scale=0.3)
    a, b, c = (v.detach().clone().requires_grad_() for _ in range(3))
    dy = make(rows, rows, t=FP, seed=3, grad=False)
    once = torch.autograd.grad(
        gt.linear_act(v, v, None, v, act="silu"), v, dy)[0]
    parts = torch.autograd.grad(
        gt.linear_act(a, b, None, c, act="silu"), (a, b, c), dy)
    # two additions of three values in fp32
    bound = sum(p.abs() for p in parts) * 2 ** -22
    assert bool(((once - sum(parts)).abs() <= bound).all())


@pytest.mark.parametrize("act8", [False, True])
@pytest.mark.parametrize("rows", [3, 150])
def test_block_gradients_that_are_no_plain_tensor(act8, rows):
    """A gradient expanded from one value, a transposed one, a graph kept for a
    second pass, and gradients that add up."""
    args = block_args(rows, 72, 200, BF)
    y = gt.ffn_block(*args, act8=act8)
    flat = torch.autograd.grad(y, args, torch.ones_like(y), retain_graph=True)
    wide = torch.autograd.grad(y, args, y.new_ones(()).expand(y.shape),
                               retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(flat, wide))
    dy = make(72, rows, t=BF, seed=8, grad=False)
    turned = torch.autograd.grad(y, args, dy.t(), retain_graph=True)
    whole = torch.autograd.grad(y, args, dy.t().contiguous(),
                                retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(turned, whole))
    y.backward(dy.t(), retain_graph=True)
    assert all(torch.equal(p.grad, b) for p, b in zip(args, whole))
    y.backward(dy.t())
    for p, b in zip(args, whole):
        assert torch.equal(p.grad, 2 * b)


@pytest.mark.parametrize("rows", [7, 200])
@pytest.mark.parametrize("t", [BF, HF, FP])
def test_block_parameters_out_of_one_buffer(rows, t):
    """Parameters at every alignment that the type allows, as views of one flat
    buffer are."""
    args = block_args(rows, 39, 77, t)
    dy = make(rows, 39, t=t, seed=8, grad=False)
    want = torch.autograd.grad(gt.ffn_block(*args), args, dy)
    size = sum(a.numel() + 1 for a in args)
    flat = torch.empty(size, dtype=t, device=DEV)
    at, views = 1, []
    for a in args:
        v = flat[at:at + a.numel()].view(a.shape)
        v.copy_(a.detach())
        views.append(v.detach().requires_grad_())
        at += a.numel() + 1
    got = torch.autograd.grad(gt.ffn_block(*views), views, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_threads_at_once():
    import threading
    args = [block_args(rows, 72, 200, BF) for rows in (40, 300)]
    dys = [torch.ones_like(a[0]) for a in args]
    want = [torch.autograd.grad(gt.ffn_block(*a, act8=True), a, dy)
            for a, dy in zip(args, dys)]
    got = [None, None]
    torch.cuda.synchronize()

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got[i] = torch.autograd.grad(
                    gt.ffn_block(*args[i], act8=True), args[i], dys[i])
        s.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_other_stream():
    args = block_args(300, 200, 400, BF)
    dy = make(300, 200, t=BF, seed=9, grad=False)
    want = torch.autograd.grad(gt.ffn_block(*args, act8=True), args, dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        # work that delays this stream and not the other
        big = torch.randn(4096, 4096, device=DEV)
        for _ in range(8):
            big = big @ big * 1e-3
        late = [(a.detach() + 0 * big[0, 0].to(a.dtype)).requires_grad_(True)
                for a in args]
        got = torch.autograd.grad(gt.ffn_block(*late, act8=True), late, dy)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_steps():
    """Two captured training steps of different sizes, replayed in turn with
    eager work between them; every replay against the eager result."""
    sets = []
    for rows, act8 in ((300, True), (150, False)):
        args = block_args(rows, 120, 480, BF)
        dy = make(rows, 120, t=BF, seed=9, grad=False)

        def step(args=args, dy=dy, act8=act8):
            y = gt.ffn_block(*args, act8=act8)
            return [y.detach(), *torch.autograd.grad(y, args, dy)]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(2):
                step()
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        sets.append((args, step, graph, outs))
    for turn in range(4):
        for args, step, graph, outs in sets:
            with torch.no_grad():
                args[0].add_(0.125 * turn)
            want = step()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b)


@pytest.mark.parametrize("m,k,n,t", [(1, 100, 300, BF), (20, 1500, 700, HF),
                                     (33, 77, 50, FP), (20000, 499, 20100, BF)])
def test_captured_linear_layers(m, k, n, t):
    """Few rows, and operands that are copied to rows on lines: every replay
    against the eager result, with eager work between."""
    x, w = make(m, k, t=t), make(n, k, t=t, scale=k ** -0.5, seed=1)
    b, g = make(n, t=t, seed=2), make(k, t=t, seed=4)
    dy = make(m, n, t=t, seed=3, grad=False)

    def step():
        with torch.no_grad():
            plain = gt.linear_act(gt.layer_norm(x, g), w, b, act="silu")
        y = gt.linear_act(x, w, b)
        return [plain, y.detach(), *torch.autograd.grad(y, (x, w, b), dy)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for turn in range(3):
        with torch.no_grad():
            x.add_(0.25 * turn)
            w.mul_(1.0 + 0.5 * turn)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs, want))


@pytest.mark.parametrize("which", ["norm", "linear", "block"])
def test_capture_refuses_a_living_graph_of_its_leaves(which):
    args = block_args(40, 24, 56, BF)
    x, gamma, beta, w1, b1 = args[:5]
    call = {"norm": lambda: gt.layer_norm(x, gamma, beta),
            "linear": lambda: gt.linear_act(x, w1, b1, act="gelu"),
            "block": lambda: gt.ffn_block(*args)}[which]
    leaves = {"norm": (x, gamma, beta), "linear": (x, w1, b1),
              "block": args}[which]
    dy = torch.ones_like(call())
    want = torch.autograd.grad(call(), leaves, dy)
    living = call()
    graph = torch.cuda.CUDAGraph()
    mark = torch.zeros(1, device=DEV)
    with pytest.raises(RuntimeError, match="free that graph"):
        with torch.cuda.graph(graph):
            mark += 1
            call()
    del living, graph
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(call(), leaves, dy)
        twice = call()          # a second call of one capture is not refused
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_autocast_keeps_fp32_parameters():
    block = gt.FFNBlock(96, 192, act8=True).to(DEV)
    x = make(50, 96)
    with torch.autocast("cuda", dtype=BF):
        y = block(x)
        z = gt.FusedLinearAct(96, 33, act="relu").to(DEV)(x)
    assert y.dtype == BF and z.dtype == BF
    y.float().square().sum().backward()
    for p in block.parameters():
        assert p.grad.dtype == FP and torch.isfinite(p.grad).all()
    assert x.grad.dtype == FP


def test_refusals_gpu():
    x, w = make(3, 8, t=BF), make(5, 8, t=BF)
    with pytest.raises(RuntimeError, match="weight must be"):
        gt.linear_act(x, make(5, 8))
    with pytest.raises(RuntimeError, match="weight is on"):
        gt.linear_act(x, w.cpu())
    with pytest.raises(RuntimeError, match="weight must have shape"):
        gt.linear_act(x, make(5, 7, t=BF))
    with pytest.raises(RuntimeError, match="bias must have shape"):
        gt.linear_act(x, w, make(8, t=BF))
    with pytest.raises(RuntimeError, match="bias must be"):
        gt.linear_act(x, w, make(5, t=HF))
    with pytest.raises(RuntimeError, match="residual must have"):
        gt.linear_act(x, w, residual=make(5, t=BF))
    with pytest.raises(RuntimeError, match="residual must be"):
        gt.linear_act(x, w, residual=make(3, 5))
    with pytest.raises(RuntimeError, match="x must be"):
        gt.linear_act(x.double(), w.double())
    with pytest.raises(RuntimeError, match="weight must be"):
        gt.layer_norm(x, make(8, t=HF))
    with pytest.raises(RuntimeError, match="weight is"):
        gt.layer_norm(x, make(8), make(8, t=BF))
    with pytest.raises(RuntimeError, match="last dimension"):
        gt.layer_norm(make(3, 0, t=BF))
    with pytest.raises(RuntimeError, match="at least one dimension"):
        gt.layer_norm(x.detach()[0, 0])
    with pytest.raises(RuntimeError, match="w2 must have shape"):
        gt.ffn_block(x, None, None, make(16, 8, t=BF), None,
                     make(9, 16, t=BF), None)
    with pytest.raises(RuntimeError, match="codes must be"):
        gt.act8_unpack(x.detach(), x.detach().float())
    with pytest.raises(RuntimeError, match="scales must have"):
        gt.act8_unpack(torch.zeros(3, 200, dtype=torch.int8, device=DEV),
                       torch.zeros(3, 1, device=DEV))
    with pytest.raises(RuntimeError, match="act8_unpack gives"):
        gt.act8_unpack(torch.zeros(3, 8, dtype=torch.int8, device=DEV),
                       torch.zeros(3, 1, device=DEV), torch.float64)
    one = torch.zeros(1, 1, device=DEV)     # views of it hold no memory
    with pytest.raises(RuntimeError, match="too large"):
        gt.act8_pack(one.expand(2 ** 30, 1))
    with pytest.raises(RuntimeError, match="too large"):
        gt.linear_act(one.expand(2 ** 30, 1), one)
    with pytest.raises(RuntimeError, match="too large"):
        gt.linear_act(one.expand(1, 4000001), one.expand(1, 4000001))
    with pytest.raises(RuntimeError, match="too long"):
        gt.layer_norm(one.expand(1, 2 ** 25))
    for f in (lambda: gt.layer_norm(x), lambda: gt.linear_act(x, w)):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(f().sum(), x, create_graph=True)
    y = gt.linear_act(x, w)
    with torch.no_grad():
        w.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


@pytest.mark.parametrize("amp", [True, False])
def test_lstm_with_block_trains(amp):
    """The language model with the block, its parameters in the optimizer's
    flat buffer, where they start at any multiple of four bytes."""
    tr = DLTrainer(dnn="lstm", dataset="ptb", batch_size=5, lr=0.1,
                   device=DEV, amp=amp, num_workers=0, n_samples=64,
                   model_kwargs={"vocab_size": 121, "hidden": 25,
                                 "ffn_mult": 3, "act8": True})
    opt = gt.DistributedOptimizer(
        tr.optimizer, tr.net.named_parameters(),
        compression=gt.compressors["gtopk"](0.05), density=0.05)
    before = tr.net.ffn.fc1.weight.detach().clone()
    for _ in range(3):
        loss = tr.train(1, dist_optimizer=opt)
        tr.update_model(dist_optimizer=opt)
    assert loss == loss
    assert not torch.equal(before, tr.net.ffn.fc1.weight)
    assert "perplexity" in tr.test()


def test_lstm_block_eval_is_training_forward():
    torch.manual_seed(0)
    net = zoo.lstm_ptb(50, 24, ffn_mult=2).to(DEV).eval()
    toks = torch.randint(0, 50, (7, 3), device=DEV)
    a, _ = net(toks, net.init_hidden(3))
    with torch.no_grad():
        b, _ = net(toks, net.init_hidden(3))
    assert torch.equal(a, b)
