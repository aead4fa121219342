"""The large tiles of the weight gradient taken from 8-bit checkpoints: 64 x 256, 128 x 128 and 256 x 256 outputs, over one range of rows and over
several, with last steps of all 32 rows and of fewer, with odd numbers of outputs (pairs of columns that pass the last one), odd
row strides (pairs of 16-bit gradients at any 2-byte address) and batches of fewer rows than a step."""
import pytest
import torch

from dun_amd import act8
from tests.row_oracle import U32

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

# rows, outputs, columns: [tile] [ranges of rows] [rows of the last step]
SHAPES = [(34, 1857, 2295),     # 64 x 256, one, 2
          (17376, 39, 1255),    # 64 x 256, 50, 32
          (4845, 67, 2131),     # 64 x 256, 14, 13
          (7, 4097, 8191),      # 64 x 256, one, 7 of 7
          (644, 1487, 2589),    # 128, one, 4
          (7803, 1477, 69),     # 128, 41, 27
          (16384, 513, 513),    # 128, 20, 32
          (31, 5473, 2817),     # 128, one, 31 of 31
          (68, 2257, 3825),     # 256, one, 4
          (2000, 2047, 2049),   # 256, 3, 16
          (16384, 1001, 517),   # 256, 21, 32
          (27023, 641, 139),    # 256, 85, 15
          (8, 4097, 16383)]     # 256, one, 8 of 8


def beside_nan(t, rows_behind=5):
    """The same rows as part of a longer and wider tensor with an odd row stride, NaN all around them."""
    rows, cols = t.shape
    wide = torch.full((rows + rows_behind, cols + 5 - cols % 2), float("nan"), dtype=t.dtype, device=t.device)
    assert wide.stride(0) % 2 == 1
    wide[:rows, 1:1 + cols] = t
    return wide[:rows, 1:1 + cols]


@pytest.mark.parametrize("rows,outs,cols", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("relu", [False, True])
def test_whole_numbers_are_exact(rows, outs, cols, dtype, relu):
    """Codes of scale 1 and whole gradients so small that every sum stays below 2^24: each addition is exact in float32, in whatever order."""
    g = torch.Generator(device="cuda").manual_seed(rows + outs + cols)
    limit = 255 if relu else 127
    most = min(30, ((1 << 24) - 1) // (limit * rows))
    assert most >= 1
    x = torch.randint(-limit, limit + 1, (rows, cols), generator=g, device="cuda").float()
    x[:, ::32] = limit
    v = x.clamp(min=0).double() if relu else x.double()
    dy = torch.randint(-most, most + 1, (rows, outs), generator=g, device="cuda").to(dtype)
    d = beside_nan(dy)
    p = act8.pack(x, relu=relu)
    assert torch.equal(p.unpack().double(), v)
    dw, db = act8.weight_grad(d, p)
    assert torch.equal(dw.double(), dy.double().t() @ v) and torch.equal(db.double(), dy.double().sum(0))
    only, none = act8.weight_grad(dy, p, bias=False)
    assert none is None and torch.equal(only, dw)


def bound(d, v, rows):
    """|error| <= (2 rows + 64) u sum |dy| |value|: every addition of the float32 accumulation off by at most 2 u of a partial sum (the matrix
    cores' adders may cut off instead of rounding), in the worst order."""
    return (2 * rows + 64) * U32 * (d.abs().t() @ v.abs()) + 1e-37


@pytest.mark.parametrize("rows,outs,cols", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("relu", [False, True])
def test_gradients_of_all_their_bits(rows, outs, cols, dtype, relu):
    g = torch.Generator(device="cuda").manual_seed(rows * 3 + outs + cols)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    dy = (r(rows, outs) * torch.exp(r(rows, 1)) / rows ** 0.5).to(dtype)
    p = act8.pack(r(rows, cols), relu=relu)
    v, d = p.unpack().double(), dy.double()
    dw, db = act8.weight_grad(beside_nan(dy), p)
    want = d.t() @ v
    assert ((dw.double() - want).abs() <= bound(d, v, rows)).all()
    assert ((db.double() - d.sum(0)).abs() <= (rows + 64) * U32 * d.abs().sum(0) + 1e-37).all()
    # in the 2-norm the errors of a sum of random terms add like a random walk: 2 u a step, with room for 2
    assert (dw.double() - want).norm() <= 4 * U32 * (rows ** 0.5 + 4) * want.norm()
    again = act8.weight_grad(dy, p)
    assert torch.equal(again[0], dw) and torch.equal(again[1], db)


@pytest.mark.parametrize("rows,outs,cols", [(7803, 1477, 69), (68, 2257, 3825), (2000, 2047, 2049)])
def test_a_group_that_is_not_finite_stays_in_its_columns(rows, outs, cols):
    x = torch.randn(rows, cols, device="cuda")
    x[rows - 1, 40] = float("inf")
    dw, db = act8.weight_grad(torch.ones(rows, outs, device="cuda"), act8.pack(x))
    hit = torch.zeros(cols, dtype=torch.bool, device="cuda")
    hit[32:64] = True
    assert torch.equal(torch.isnan(dw), hit.expand(outs, cols)) and torch.equal(db, torch.full_like(db, float(rows)))


def test_captured_and_replayed_over_several_ranges():
    x, dy = torch.randn(27023, 139, device="cuda"), torch.randn(27023, 641, device="cuda")
    step = lambda: act8.weight_grad(dy, act8.pack(x))
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        x.copy_(torch.randn_like(x))
        dy.copy_(torch.randn_like(dy))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step())), k
