"""dun_amd.layer_norm on the GPU against the formulas in 64 bits (tests/row_oracle.py, where the bounds are derived)."""
import pytest
import torch

from dun_amd import act8
from dun_amd.layer_norm import LayerNorm, layer_norm, layer_norm_backward, layer_norm_forward
from tests.row_oracle import Norm, U32, codes_of, within

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# one row, one element, around every switch of the team (8 to 64 lanes of 4 or 8 elements, vectors per lane, 256 and 1024 lanes,
# rows walked in memory), many rows
SHAPES = [(1, 1), (1, 2), (3, 3), (2, 31), (5, 32), (4, 33), (9, 64), (3, 65), (33, 100), (7, 127), (2, 256), (5, 257), (3, 513),
          (2, 1023), (3, 1031), (2, 2048), (3, 2049), (2, 4099), (2, 8192), (1, 8193), (2, 16385), (1, 32768), (2, 33001), (1, 70003),
          (513, 100), (4099, 517), (20011, 7), (2500, 2047)]


def make(rows, cols, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * spread + 0.5 * torch.randn(rows, 1, generator=g)
    w = 1 + 0.3 * torch.randn(cols, generator=g)
    b = 0.2 * torch.randn(cols, generator=g)
    res = torch.randn(rows, cols, generator=g)
    dy = torch.randn(rows, cols, generator=g)
    return x.to(dtype).cuda(), w.cuda(), b.cuda(), res.to(dtype).cuda(), dy.to(dtype).cuda()


def check(x, w, b, eps, res, relu, bits, dy, sum_dx=True):
    o = Norm(x, w, b, eps, res, relu, bits).backward(dy)
    y, saved = layer_norm_forward(x, w, b, eps, residual=res, relu=relu, bits=bits)
    within(y, o.y, o.y_tol, "y")
    out = layer_norm_backward(dy, saved, sum_dx=sum_dx)
    within(out[0], o.dx, o.dx_tol, "dx")
    within(out[1], o.dw, o.dw_tol, "dw")
    within(out[2], o.db, o.db_tol, "db")
    if sum_dx:
        # (the sum takes dx before its rounding to the type)
        within(out[3], o.ds, o.ds_tol, "sum dx")
    return y, out


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_forward_backward(rows, cols, dtype):
    x, w, b, res, dy = make(rows, cols, dtype, rows * 7 + cols)
    check(x, w, b, 1e-5, None, False, None, dy, sum_dx=False)


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_residual_block_from_the_checkpoint(rows, cols, dtype):
    x, w, b, res, dy = make(rows, cols, dtype, rows * 11 + cols)
    check(x, w, b, 1e-5, res, True, 8, dy)


@pytest.mark.parametrize("rows,cols", [(3, 1), (5, 33), (64, 100), (3, 2049), (2, 9000), (1, 33001)])
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("affine", ["none", "weight", "bias"])
def test_combinations(rows, cols, relu, bits, affine):
    x, w, b, res, dy = make(rows, cols, F32, rows + cols, spread=3.0)
    w = w if affine == "weight" else None
    b = b if affine == "bias" else None
    check(x, w, b, 1e-3, res if relu else None, relu, bits, dy)
    y = layer_norm(x, w, b, 1e-3, res, relu)  # without anything kept
    o = Norm(x, w, b, 1e-3, res, relu)
    within(y, o.y, o.y_tol, "y")


def test_rows_far_from_zero_lose_nothing():
    # mean 1000 spreads: squares of sums would cancel, squares of differences do not
    x, w, b, res, dy = make(64, 300, F32, 3, spread=1e-2)
    check(x + 10.0, w, b, 1e-12, None, False, None, dy)


def test_constant_rows():
    x = torch.full((5, 77), 3.25, device="cuda")
    y, saved = layer_norm_forward(x, None, None, 1e-5)
    assert torch.equal(y, torch.zeros_like(y))
    dx, dw, db = layer_norm_backward(torch.ones_like(x), saved)
    assert torch.isfinite(dx).all() and torch.equal(dw, torch.zeros_like(dw)) and torch.equal(db, torch.full_like(db, 5.0))


@pytest.mark.parametrize("bits", [None, 8])
def test_all_rows_dead_under_relu(bits):
    x = -torch.rand(9, 130, device="cuda") - 0.1
    res = torch.randn(9, 130, device="cuda")
    y, saved = layer_norm_forward(x, None, None, 1e-5, residual=res, relu=True, bits=bits)
    assert torch.equal(y, res)
    dx = layer_norm_backward(torch.randn_like(x), saved)[0]
    assert torch.equal(dx, torch.zeros_like(dx))


@pytest.mark.parametrize("bits", [None, 8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("cols", [70, 3001, 40000])
def test_a_bad_row_stays_its_own(bits, bad, cols):
    x, w, b, res, dy = make(6, cols, F32, 5)
    x[2, cols // 2] = bad
    y, saved = layer_norm_forward(x, w, b, 1e-5, residual=res, bits=bits)
    dx, dw, db = layer_norm_backward(dy, saved)
    keep = [0, 1, 3, 4, 5]
    o = Norm(x[keep], w, b, 1e-5, res[keep], False, bits).backward(dy[keep])
    within(y[keep], o.y, o.y_tol, "y")
    within(dx[keep], o.dx, o.dx_tol, "dx")
    assert not torch.isfinite(y[2]).any() and not torch.isfinite(dx[2]).any() and not torch.isfinite(dw).any()
    assert torch.isfinite(db).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_orders(dtype):
    g = torch.Generator().manual_seed(9)
    wide = torch.randn(40, 301, generator=g).to(dtype).cuda()
    w, b = torch.randn(97, generator=g).cuda(), torch.randn(97, generator=g).cuda()
    x, res = wide[:, 3:100], wide[:, 150:247]                       # rows of a wider tensor, unaligned
    dy = torch.randn(97, 40, generator=g).to(dtype).cuda().t()     # columns as rows: copied
    assert x.stride() == (301, 1) and dy.stride() == (1, 40)
    before = wide.clone()
    check(x, w, b, 1e-5, res, True, 8, dy)
    check(x, w, b, 1e-5, res, False, None, dy)
    check(wide[::3, 5:102], w, b, 1e-5, None, False, None, dy[:14])
    one = torch.randn(1, 97, generator=g).to(dtype).cuda().expand(40, 97)  # broadcast rows
    check(one, w, b, 1e-5, None, False, None, one)
    assert torch.equal(wide, before)


def test_more_dimensions_and_empty():
    x = torch.randn(3, 5, 7, 33, device="cuda", requires_grad=True)
    y = layer_norm(x)
    assert y.shape == x.shape
    assert torch.allclose(y, torch.nn.functional.layer_norm(x, (33,)), atol=1e-5)
    v = layer_norm(torch.randn(33, device="cuda"))
    assert v.shape == (33,)
    w = torch.randn(33, device="cuda", requires_grad=True)
    e = torch.empty(0, 33, device="cuda", requires_grad=True)
    for bits in (None, 8):
        gx, gw = torch.autograd.grad(layer_norm(e, w, bits=bits).sum(), (e, w))
        assert gx.shape == (0, 33) and torch.equal(gw, torch.zeros_like(w))


def test_autograd_matches_the_halves_and_torch():
    x, w, b, res, dy = make(50, 200, F32, 21)
    for t in (x, w, b, res):
        t.requires_grad_()
    y = layer_norm(x, w, b, 1e-5, residual=res)
    got = torch.autograd.grad(y, (x, w, b, res), dy)
    ref = torch.autograd.grad(torch.nn.functional.layer_norm(x.double(), (200,), w.double(), b.double()) + res.double(),
                              (x, w, b, res), dy.double())
    for a, c in zip(got, ref):
        assert torch.allclose(a, c.float(), rtol=1e-4, atol=1e-5)
    _, saved = layer_norm_forward(x, w, b, 1e-5, residual=res)
    halves = layer_norm_backward(dy, saved)
    assert all(torch.equal(a, c) for a, c in zip(got, halves)) and torch.equal(got[3], dy)


def test_gradient_against_differences():
    x, w, b, res, dy = make(4, 37, F32, 22)
    for t in (x, w, b):
        t.requires_grad_()
    z = layer_norm(x, w, b, 1e-5, residual=res, relu=True)
    gx, gw, gb = torch.autograd.grad(z, (x, w, b), dy)
    # along a direction, central differences of the 64-bit formula: error O(h^2)
    g = torch.Generator().manual_seed(1)
    h = 1e-5
    for t, grad in ((x, gx), (w, gw), (b, gb)):
        d = torch.randn(t.shape, generator=g, dtype=torch.float64)

        def loss(s):
            args = {id(u): u.detach().cpu().double() for u in (x, w, b)}
            args[id(t)] = args[id(t)] + s * d
            zz = torch.relu(args[id(x)])
            m = zz.mean(1, keepdim=True)
            v = ((zz - m) ** 2).mean(1, keepdim=True)
            return float((((zz - m) / torch.sqrt(v + 1e-5) * args[id(w)] + args[id(b)]) * dy.cpu().double()).sum())

        slope = (loss(h) - loss(-h)) / (2 * h)
        along = float((grad.cpu().double() * d).sum())
        assert abs(slope - along) <= 1e-4 * (1 + float((grad.cpu().double() * d).abs().sum()))


@pytest.mark.parametrize("wtype", [F32, BF16, F16])
def test_weight_types(wtype):
    x, w, b, res, dy = make(65, 96, BF16, 23)
    w, b = w.to(wtype).requires_grad_(), b.to(wtype).requires_grad_()
    o = Norm(x, w, b, 1e-5).backward(dy)
    y = layer_norm(x.requires_grad_(), w, b, 1e-5)
    within(y, o.y, o.y_tol, "y")
    gw, gb = torch.autograd.grad(y, (w, b), dy)
    assert gw.dtype == gb.dtype == wtype
    half = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}[wtype]
    within(gw, o.dw, o.dw_tol + half * o.dw.abs() + half * 1e-3, "dw")
    within(gb, o.db, o.db_tol + half * o.db.abs() + half * 1e-3, "db")


def test_the_kept_checkpoint_and_the_packed_output():
    x, w, b, res, dy = make(37, 517, F32, 24)
    y, saved, packed = layer_norm_forward(x, w, b, 1e-5, residual=res, relu=True, bits=8, pack_output=True)
    q, e = codes_of(x, True)
    assert torch.equal(saved.packed[0].cpu().double().view(q.shape), q) and torch.equal(saved.packed[1].cpu().double(), e + 127)
    q, e = codes_of(y, False)
    assert torch.equal(packed.codes.cpu().double().view(q.shape) - 128, q)
    alone = act8.pack(y)
    assert torch.equal(alone.codes, packed.codes) and torch.equal(alone.exps, packed.exps)
    for dtype in (BF16, F16):
        y, _, packed = layer_norm_forward(x.to(dtype), w, b, 1e-5, pack_output=True)
        alone = act8.pack(y)
        assert torch.equal(alone.codes, packed.codes) and torch.equal(alone.exps, packed.exps)


def test_same_bits_every_time():
    x, w, b, res, dy = make(5001, 257, F32, 25)
    first = None
    for _ in range(3):
        y, saved = layer_norm_forward(x, w, b, 1e-5, res, True, 8)
        out = (y,) + layer_norm_backward(dy, saved, sum_dx=True)
        first = first or out
        assert all(torch.equal(a, c) for a, c in zip(first, out))


def test_module():
    m = LayerNorm(100, bits=8).cuda()
    ref = torch.nn.LayerNorm(100).cuda()
    ref.load_state_dict(m.state_dict())
    x = torch.randn(20, 100, device="cuda")
    assert torch.allclose(m(x), ref(x), atol=1e-5)
    m(x).square().sum().backward()
    assert m.weight.grad is not None and m.bias.grad is not None


def test_captured_and_replayed():
    x, w, b, res, dy = make(300, 100, F32, 26)
    dx_in = dy.clone()

    def step():
        y, saved = layer_norm_forward(x, w, b, 1e-5, res, True, 8)
        return (y,) + layer_norm_backward(dx_in, saved, sum_dx=True)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        x.copy_(torch.randn(300, 100, device="cuda"))
        dx_in.copy_(torch.randn(300, 100, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, c) for a, c in zip(held, want)), k


def test_on_another_stream():
    x, w, b, res, dy = make(2000, 513, F32, 27)
    want, saved = layer_norm_forward(x, w, b, 1e-5, res, True, 8)
    want = (want,) + layer_norm_backward(dy, saved)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, saved = layer_norm_forward(x, w, b, 1e-5, res, True, 8)
        got = (y,) + layer_norm_backward(dy, saved)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_more_than_2_31_elements():
    rows, cols = 1_100_000, 2000  # 2.2e9 elements
    x = torch.zeros(rows, cols, device="cuda", dtype=BF16)
    x[-3:] = torch.randn(3, cols, device="cuda").to(BF16)
    y, saved, packed = layer_norm_forward(x, None, None, 1e-5, relu=True, bits=8, pack_output=True)
    o = Norm(x[-3:], None, None, 1e-5, None, True, 8).backward(x[-3:])
    within(y[-3:], o.y, o.y_tol, "y")
    assert not y[:-3].any()
    q, _ = codes_of(x[-3:], True)
    assert torch.equal(saved.packed[0][-3:].cpu().double().view(q.shape), q)
    dx, dw, db = layer_norm_backward(x, saved)
    within(dx[-3:], o.dx, o.dx_tol, "dx")
    within(dw, o.dw, o.dw_tol * 4, "dw")  # (the other rows add exact zeros)


@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 33), (300, 100), (40, 1031), (9, 9000)])
@pytest.mark.parametrize("bits", [None, 8])
def test_dx_alone(rows, cols, bits):
    x, w, b, res, dy = make(rows, cols, F32, 31)
    o = Norm(x, w, b, 1e-5, res, True, bits).backward(dy)
    y = layer_norm(x.requires_grad_(), w, b, 1e-5, res, True, bits)
    within(torch.autograd.grad(y, x, dy, retain_graph=True)[0], o.dx, o.dx_tol, "dx")
    r2 = res.clone().requires_grad_()
    y = layer_norm(x.detach(), w, b, 1e-5, r2, True, bits)
    assert torch.equal(torch.autograd.grad(y, r2, dy)[0], dy)


def test_output_in_place_of_the_residual_and_gradient_in_place():
    from dun_amd import kernels
    be = kernels.backend()
    for cols in (3, 33, 1031, 2049, 9001):
        x, w, b, res, dy = make(50, cols, F32, cols)
        want, saved = layer_norm_forward(x, w, b, 1e-5, res, True)
        dx = layer_norm_backward(dy, saved)[0]
        y, stats, _, _ = be.layer_norm_forward(x, w, b, 1e-5, res, True, out=res)
        got, _ = be.layer_norm_backward(dy, x, None, w, stats, True, 2, dx=dy)
        assert torch.equal(y, want) and torch.equal(got, dx)


def test_autograd_under_capture():
    x, w, b, res, dy = make(128, 200, F32, 33)
    leaves = [t.requires_grad_() for t in (x, w, b, res)]

    def step():
        y = layer_norm(*leaves[:3], 1e-5, leaves[3], True, 8)
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(held, step()))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("relu", [False, True])
def test_rows_of_one_element(dtype, relu):
    # the element is its own mean: y = bias, and g - mean(g) = 0 exactly whatever the rounding of g = dy weight is
    x = torch.randn(37, 1, device="cuda").to(dtype)
    dy = torch.randn(37, 1, device="cuda").to(dtype)
    w, b = torch.tensor([1.1], device="cuda"), torch.tensor([0.375], device="cuda")
    y, saved = layer_norm_forward(x, w, b, 1e-5, relu=relu)
    dx, dw, db, ds = layer_norm_backward(dy, saved, sum_dx=True)
    assert torch.equal(y, torch.full_like(y, 0.375))
    assert torch.equal(dx, torch.zeros_like(dx)) and torch.equal(dw, torch.zeros_like(dw)) and torch.equal(ds, torch.zeros_like(ds))
    within(db, dy.double().cpu().sum(0), 128 * U32 * dy.double().cpu().abs().sum(0), "db")


@pytest.mark.parametrize("cols", [7, 100, 517, 2048, 9000])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_row_that_is_not_finite_has_no_gradient_anywhere(cols, bad):
    x, w, b, _, dy = make(3, cols, F32, 7)
    x[1, cols // 2] = bad
    _, saved = layer_norm_forward(x, w, b, 1e-5)
    for kw in ({}, {"sum_dx": True}, {"weight_grads": False}):
        dx = layer_norm_backward(dy, saved, **kw)[0]
        assert torch.isnan(dx[1]).all() and torch.isfinite(dx[0]).all() and torch.isfinite(dx[2]).all(), kw
