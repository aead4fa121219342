"""dun_amd.act8 on the GPU: codes against the definition (exactly), gradients against 64-bit products of the values."""
import pytest
import torch

from dun_amd import act8, kernels
from dun_amd.layer_norm import layer_norm
from tests.row_oracle import U32, codes_of, values_of, within

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SHAPES = [(1, 1), (3, 2), (2, 31), (4, 32), (5, 33), (7, 95), (64, 100), (3, 1001), (2, 4097), (513, 517), (3000, 2048)]


def rand(*shape, seed=0, spread=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * spread


def same_codes(packed, x, relu):
    q, e = codes_of(x, relu)
    zero = 0 if relu else 128
    assert torch.equal(packed.codes.cpu().double().view(q.shape) - zero, q)
    assert torch.equal(packed.exps.cpu().double(), e + 127)
    v = values_of(x, relu)
    got = packed.unpack().cpu().double()
    assert torch.equal(torch.nan_to_num(got, 7e30), torch.nan_to_num(v, 7e30))


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("relu", [False, True])
def test_codes_and_values(rows, cols, dtype, relu):
    x = rand(rows, cols, seed=rows + cols) * torch.exp(3 * rand(rows, 1, seed=1))
    x = x.to(dtype).cuda()
    p = act8.pack(x, relu=relu)
    same_codes(p, x, relu)
    assert p.nbytes == p.codes.numel() + p.exps.numel() and p.shape == (rows, cols)
    # off by at most half a step; a positive rectified element is at least one step (the spread of the rows overflows
    # float16 in some: a group with an infinity reads back as NaN, checked above)
    step = torch.exp2(p.exps.cpu().double() - 127).repeat_interleave(32, dim=1)[:, :cols]
    v, z = p.unpack().cpu().double(), x.cpu().double()
    z = z.clamp(min=0) if relu else z
    fine = torch.isfinite(v)
    assert ((v - z).abs() <= (step if relu else step / 2))[fine].all()
    assert torch.equal((v > 0)[fine], (z > 0)[fine]) if relu else True


@pytest.mark.parametrize("relu", [False, True])
def test_scales_at_their_borders(relu):
    # largest magnitudes next to where the scale changes, at every exponent, zero and denormal groups
    limit = 255.5 if relu else 127.5
    tops = []
    for k in list(range(-149, 121, 3)) + [119, 120]:
        for m in (limit, limit * (1 - 2.0 ** -23), limit * (1 + 2.0 ** -23), 64.0, 128.0, 127.0, 255.0, 1.0):
            tops.append(m * 2.0 ** k)
    tops += [0.0, 2.0 ** -149, 2.0 ** -126, 3.4028234663852886e38, 1.7e38, 2.0 ** 127]
    tops = [t for t in tops if t < 3.4028235e38]
    x = rand(len(tops), 64, seed=4).clamp(-1, 1)
    x = (x.double() * torch.tensor(tops, dtype=torch.float64).view(-1, 1)).float()
    x[:, 5] = torch.tensor(tops, dtype=torch.float64).float()
    x[:, 40] = x[:, 5]
    x = x.cuda()
    same_codes(act8.pack(x, relu=relu), x, relu)


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_groups_that_are_not_finite(relu, bad):
    x = rand(4, 96, seed=5).cuda()
    x[1, 40] = bad
    p = act8.pack(x, relu=relu)
    v = p.unpack()
    hit = torch.zeros(4, 96, dtype=torch.bool)
    hit[1, 32:64] = not (relu and bad == float("-inf"))
    assert torch.equal(torch.isnan(v).cpu(), hit)
    same_codes(p, x, relu)
    dw, db = act8.weight_grad(torch.ones(4, 3, device="cuda"), p)
    assert torch.equal(torch.isnan(dw).cpu(), hit[1].expand(3, 96))
    assert torch.equal(db, torch.full((3,), 4.0, device="cuda"))


def test_strides_types_and_shapes_of_unpack():
    wide = rand(20, 203, seed=6).cuda()
    for x in (wide[:, 3:100], wide.t(), wide[::2, 100:101], rand(1, 33, seed=7).cuda().expand(9, 33)):
        same_codes(act8.pack(x), x, False)
    x = rand(2, 3, 5, 40, seed=8).cuda()
    p = act8.pack(x)
    v = p.unpack()
    assert v.shape == x.shape
    assert torch.equal(p.unpack(BF16).float(), v)          # a value is a bf16 number
    assert torch.equal(p.unpack(F16), v.to(F16))
    assert act8.pack(torch.empty(0, 5, device="cuda")).unpack().shape == (0, 5)


def grad_bound(dy, v, rows):
    """|error| <= (rows + 64) u sum |dy| |value|: every addition of the fp32 accumulation off by at most 2 u of a partial sum (the
    matrix cores' adders may cut off instead of rounding), in the worst order; and in the 2-norm 4 u (sqrt(rows) + 4): the
    errors of a sum of random terms add like a random walk."""
    return (2 * rows + 64) * U32 * (dy.abs().t() @ v.abs()) + 1e-37


@pytest.mark.parametrize("rows,outs,cols", [(1, 1, 1), (1, 7, 33), (2, 16, 32), (15, 17, 31), (16, 10, 100), (31, 33, 65), (33, 100, 100),
                                            (64, 64, 64), (100, 1, 517), (129, 300, 70), (512, 100, 100), (777, 130, 257), (1000, 10, 2048),
                                            (1024, 256, 256), (2049, 513, 300), (3000, 257, 513), (5000, 2, 40), (4096, 2048, 16),
                                            (2000, 32, 999), (2000, 31, 1024), (40000, 3, 64)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("relu", [False, True])
def test_weight_grad(rows, outs, cols, dtype, relu):
    x = rand(rows, cols, seed=rows + cols).cuda()
    dy = (rand(rows, outs, seed=outs) * torch.exp(rand(rows, 1, seed=2)) / rows ** 0.5).to(dtype).cuda()
    p = act8.pack(x, relu=relu)
    v, d = p.unpack().cpu().double(), dy.cpu().double()
    dw, db = act8.weight_grad(dy, p)
    assert dw.dtype == db.dtype == F32
    want = d.t() @ v
    within(dw, want, grad_bound(d, v, rows), "dw")
    within(db, d.sum(0), (rows + 64) * U32 * d.abs().sum(0) + 1e-37, "db")
    assert (dw.cpu().double() - want).norm() <= 4 * U32 * (rows ** 0.5 + 4) * want.norm() + 1e-30
    only, none = act8.weight_grad(dy, p, bias=False)
    assert none is None and torch.equal(only, dw)


def test_weight_grad_is_exact_where_sums_are():
    # whole numbers: codes of scale 1, gradients of up to 24 bits that take all three parts; every sum below 2^24
    rows, outs, cols = 700, 65, 96
    g = torch.Generator().manual_seed(11)
    x = torch.randint(-127, 128, (rows, cols), generator=g).float()
    x[:, ::32] = 127.0
    dy = torch.randint(-30, 31, (rows, outs), generator=g).float()
    dw, db = act8.weight_grad(dy.cuda(), act8.pack(x.cuda()))
    assert torch.equal(dw.cpu().double(), dy.double().t() @ x.double()) and torch.equal(db.cpu().double(), dy.double().sum(0))
    # one row of 24-bit numbers against powers of two: each product is the number itself, shifted
    big = torch.randint(1, 1 << 24, (1, outs), generator=g).float()
    one = torch.zeros(1, cols)
    one[0, ::32], one[0, 7::32] = 64.0, 1.0
    dw, db = act8.weight_grad(big.cuda(), act8.pack(one.cuda()))
    assert torch.equal(dw.cpu().double(), big.double().t() @ one.double()) and torch.equal(db.cpu(), big[0])


def test_weight_grad_of_extreme_magnitudes():
    x = rand(64, 64, seed=12)
    p = act8.pack((x * 1e38).clamp(-3e38, 3e38).cuda())
    v = p.unpack().cpu().double()
    dy = rand(64, 5, seed=13, spread=1e-30)
    dw, _ = act8.weight_grad(dy.cuda(), p)
    within(dw, dy.double().t() @ v, grad_bound(dy.double(), v, 64), "dw")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_weight_grad_strides(dtype):
    wide = rand(300, 77, seed=14).to(dtype).cuda()
    x = rand(300, 50, seed=15).cuda()
    p = act8.pack(x)
    v = p.unpack().cpu().double()
    for dy in (wide[:, 1:4], wide[:, 5:70], wide[:, 3:36], rand(40, 300, seed=16).to(dtype).cuda().t(), wide[:1, :9].expand(300, 9)):
        dw, db = act8.weight_grad(dy, p)
        d = dy.cpu().double()
        within(dw, d.t() @ v, grad_bound(d, v, 300), "dw")
        within(db, d.sum(0), 364 * U32 * d.abs().sum(0), "db")


def test_weight_grad_of_no_rows_and_of_more_dimensions():
    p = act8.pack(torch.empty(0, 40, device="cuda"))
    dw, db = act8.weight_grad(torch.empty(0, 6, device="cuda"), p)
    assert torch.equal(dw, torch.zeros(6, 40, device="cuda")) and torch.equal(db, torch.zeros(6, device="cuda"))
    x, dy = rand(4, 25, 40, seed=17).cuda(), rand(4, 25, 6, seed=18).cuda()
    a = act8.weight_grad(dy, act8.pack(x))
    b = act8.weight_grad(dy.reshape(100, 6), act8.pack(x.reshape(100, 40)))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_weight_grad_same_bits_every_time_and_nothing_written_past_the_end():
    dy, p = rand(4001, 70, seed=19).cuda(), act8.pack(rand(4001, 130, seed=20).cuda())
    first = act8.weight_grad(dy, p)
    for _ in range(3):
        again = act8.weight_grad(dy, p)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("bias", [True, False])
def test_linear(bias):
    x = rand(7, 30, 65, seed=21).cuda().requires_grad_()
    layer = act8.Linear(65, 33, bias=bias).cuda()
    dy = rand(7, 30, 33, seed=22).cuda()
    y = layer(x)
    want = torch.nn.functional.linear(x.double(), layer.weight.double(), None if layer.bias is None else layer.bias.double())
    assert torch.allclose(y.double(), want, atol=1e-5)
    params = [x, layer.weight] + ([layer.bias] if bias else [])
    got = torch.autograd.grad(y, params, dy)
    v = act8.pack(x).unpack().reshape(-1, 65).cpu().double()
    d = dy.reshape(-1, 33).cpu().double()
    assert torch.allclose(got[0].double(), dy.double() @ layer.weight.double(), atol=1e-4)
    within(got[1], d.t() @ v, grad_bound(d, v, 210), "dw")
    if bias:
        within(got[2], d.sum(0), 274 * U32 * d.abs().sum(0), "db")
    # dw is near the one of the unrounded input: a step is at most a 63.75th of the group's largest magnitude
    full = d.t() @ x.detach().reshape(-1, 65).cpu().double()
    assert (got[1].cpu().double() - full).norm() <= 0.02 * full.norm()


def test_linear_after_layer_norm_shares_the_checkpoint():
    x = rand(200, 96, seed=23).cuda().requires_grad_()
    w1 = torch.ones(96, device="cuda", requires_grad=True)
    layer = act8.Linear(96, 40).cuda()
    dy = rand(200, 40, seed=24).cuda()
    y, packed = layer_norm(x, w1, None, relu=True, bits=8, pack_output=True)
    a = torch.autograd.grad(layer(y, packed), (x, w1, layer.weight, layer.bias), dy)
    y = layer_norm(x, w1, None, relu=True, bits=8)
    b = torch.autograd.grad(layer(y), (x, w1, layer.weight, layer.bias), dy)
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_captured_and_replayed():
    x, dy = rand(900, 70, seed=25).cuda(), rand(900, 33, seed=26).cuda()

    def step():
        p = act8.pack(x, relu=True)
        return act8.weight_grad(dy, p) + (p.unpack(),)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        x.copy_(torch.randn(900, 70, device="cuda"))
        dy.copy_(torch.randn(900, 33, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step())), k


def test_two_graphs_share_nothing():
    a, b = rand(3000, 64, seed=27).cuda(), rand(3000, 64, seed=28).cuda()
    dy = rand(3000, 64, seed=29).cuda()
    pa, pb = act8.pack(a), act8.pack(b)
    want = act8.weight_grad(dy, pa), act8.weight_grad(dy, pb)
    torch.cuda.synchronize()
    graphs, held = [], []
    for p in (pa, pb):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(act8.weight_grad(dy, p))
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(s, t) for h, w in zip(held, want) for s, t in zip(h, w))


def test_more_than_2_31_elements():
    rows, cols = 1_100_000, 2000
    x = torch.zeros(rows, cols, device="cuda", dtype=BF16)
    x[-2:] = torch.randn(2, cols, device="cuda").to(BF16)
    p = act8.pack(x)
    q, e = codes_of(x[-2:], False)
    assert torch.equal(p.codes[-2:].cpu().double().view(q.shape) - 128, q)
    assert bool((p.codes[:-2] == 128).all())
    dy = torch.zeros(rows, 5, device="cuda")
    dy[-2:] = torch.randn(2, 5, device="cuda")
    dw, db = act8.weight_grad(dy, p)
    d, v = dy[-2:].cpu().double(), values_of(x[-2:], False)
    within(dw, d.t() @ v, grad_bound(d, v, 2), "dw")
    assert torch.equal(p.unpack(BF16)[-2:].cpu().double(), v)


@pytest.mark.parametrize("outs", [3, 40])
def test_weight_grad_of_tiny_gradients(outs):
    # a part of dy that is below bf16's smallest number, 2^-133, is lost, no more: |error| <= 2^-133 |value| on top of rounding
    v = torch.full((1, 32), 2.0 ** 100)
    p = act8.pack(v.cuda())
    for k in (-100, -110, -118, -125):
        dy = (1 + rand(1, outs, seed=30).abs()) * 2.0 ** k
        dw, _ = act8.weight_grad(dy.cuda(), p)
        want = dy.double().t() @ v.double()
        within(dw, want, 4 * U32 * want.abs() + 2.0 ** -133 * 2.0 ** 100, "dw at 2^%d" % k)


def test_weight_grad_keeps_out_what_lies_behind_the_rows():
    # rows of a longer tensor, NaN behind them and beside them: neither is read into the result
    for rows in (1, 5, 31, 33, 70, 95, 1000):
        big = torch.full((rows + 40, 60), float("nan"), device="cuda")
        big[:rows, 4:50] = rand(rows, 46, seed=rows).cuda()
        x = torch.full((rows + 40, 70), float("nan"), device="cuda")
        x[:rows] = rand(rows, 70, seed=31).cuda()
        whole = act8.pack(x)
        p = act8.Packed8(whole.codes[:rows], whole.exps[:rows], (rows, 70), False, F32)
        for dy in (big[:rows, 4:50], big[:rows, 10:13]):
            dw, db = act8.weight_grad(dy, p)
            d, v = dy.cpu().double(), p.unpack().cpu().double()
            within(dw, d.t() @ v, grad_bound(d, v, rows), "dw")
            within(db, d.sum(0), (rows + 64) * U32 * d.abs().sum(0) + 1e-37, "db")


@pytest.mark.parametrize("outs", [3, 40, 300])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_weight_grad_of_gradients_that_are_not_finite(outs, dtype, bad):
    # an infinity counts as NaN (bfloat16, which is not taken apart: as itself); only its own output sees it, and the bias exactly
    x = rand(70, 40, seed=32)
    x[33, 5] = 0
    dy = rand(70, outs, seed=33).to(dtype)
    dy[33, 1] = bad
    p = act8.pack(x.cuda())
    dw, db = act8.weight_grad(dy.cuda(), p)
    d, v = dy.double(), p.unpack().cpu().double()
    want = bad * v[33] if dtype == BF16 else torch.full((40,), float("nan"), dtype=torch.float64)
    as_numbers = lambda t: torch.nan_to_num(t.cpu().double(), 7.0, 8.0, 9.0)
    assert torch.equal(as_numbers(dw[1]), as_numbers(want))
    assert torch.equal(as_numbers(db[1]), as_numbers(torch.tensor(bad)))
    rest = [o for o in range(outs) if o != 1]
    within(dw[rest], d[:, rest].t() @ v, grad_bound(d[:, rest], v, 70), "dw")
    within(db[rest], d[:, rest].sum(0), (70 + 64) * U32 * d[:, rest].abs().sum(0) + 1e-37, "db")


def test_linear_packs_only_what_a_backward_reads(monkeypatch):
    x, layer = rand(64, 48, seed=34).cuda(), act8.Linear(48, 20).cuda()
    want = layer(x)
    calls = []
    pack = kernels.HipBackend.act8_pack
    monkeypatch.setattr(kernels.HipBackend, "act8_pack", lambda *a, **k: (calls.append(1), pack(*a, **k))[1])
    with torch.no_grad():
        assert torch.equal(layer(x), want) and not calls
    with torch.inference_mode():
        assert torch.equal(layer(x), want) and not calls
    frozen = act8.linear(x.clone().requires_grad_(), layer.weight.detach(), layer.bias.detach())
    frozen.sum().backward()
    assert torch.equal(frozen, want) and not calls
    layer(x).sum().backward()
    assert len(calls) == 1
