"""What the row operators' entries leave alone: every output and every workspace lies inside a larger buffer of a known byte, at the least
alignment that the entries take, workspaces of exactly the stated size, rows of outputs apart from each other; whatever is not
the output's own has to be that byte afterwards.  The outputs themselves have to be those of an ordinary call."""
import pytest
import torch

from dun_amd import _lib as L
from dun_amd import kernels

pytestmark = pytest.mark.gpu
F32, BF16, F16, U8 = torch.float32, torch.bfloat16, torch.float16, torch.uint8
KINDS = [F32, BF16, F16]
BYTE, PAD = 0xA5, 4096


class Guarded(object):
    """rows x cols elements, `ld` apart, `shift` elements behind an aligned address, PAD bytes around them."""

    def __init__(self, rows, cols, dtype, ld=None, shift=1):
        ld = cols if ld is None else ld
        size = dtype.itemsize
        front = PAD + shift * size
        n = (rows - 1) * ld + cols if rows else 0
        self.bytes = torch.full((front + n * size + PAD,), BYTE, dtype=U8, device="cuda")
        self.view = self.bytes[front:front + n * size].view(dtype).as_strided((rows, cols), (ld, 1), front // size)
        own = torch.zeros_like(self.bytes, dtype=torch.bool)
        own.as_strided((rows, cols * size), (ld * size, 1), front).fill_(True)
        self.others, self.ld = ~own, ld

    @property
    def p(self):
        return self.view.data_ptr()

    def check(self, want, what):
        assert bool((self.bytes[self.others] == BYTE).all()), what + ": written beside the output"
        if want is not None:
            got, want = self.view.contiguous(), want.reshape(self.view.shape).contiguous()
            assert torch.equal(got.view(U8), want.view(U8)), what


def groups(cols):
    return (cols + 31) // 32


def checkpoint(rows, cols):
    """Guarded codes (8-byte aligned and no more) and exponents."""
    return Guarded(rows, 32 * groups(cols), U8, shift=8), Guarded(rows, groups(cols), U8)


def ran(rc, what):
    L.check(rc, what)
    torch.cuda.synchronize()


def stream():
    return L.raw_stream(0)


ROWS = [(1, 1), (3, 2), (5, 3), (9, 33), (1500, 33), (7, 100), (70, 517), (4000, 517), (9, 1031), (700, 1031), (2, 4100), (3, 9001), (300, 9001)]


def make(rows, cols, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows + cols)
    return torch.randn(rows, cols, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("rows,cols", ROWS)
@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("relu,res,keep", [(False, False, False), (True, True, True), (True, False, True)])
def test_layer_norm_forward(rows, cols, dtype, relu, res, keep):
    x, r = make(rows, cols, dtype), make(rows, cols, dtype, 1) if res else None
    w, b = make(1, cols, F32, 2)[0], make(1, cols, F32, 3)[0]
    y, stats, xq, yq = kernels.backend().layer_norm_forward(x, w, b, 1e-5, r, relu, True, keep, keep)
    gy, gs = Guarded(rows, cols, dtype, ld=cols + 7), Guarded(2, rows, F32)
    (xc, xe), (yc, ye) = checkpoint(rows, cols), checkpoint(rows, cols)
    ran(L.lib().dun_layer_norm_forward(
        x.data_ptr(), cols, None if r is None else r.data_ptr(), cols, w.data_ptr(), b.data_ptr(), gy.p, gy.ld, gs.p, xc.p if keep else None,
        xe.p if keep else None, yc.p if keep else None, ye.p if keep else None, rows, cols, L.ROW_DTYPES[dtype], 1e-5, relu, stream()), "forward")
    gy.check(y, "y")
    gs.check(stats, "stats")
    for g, want, what in ((xc, xq and xq[0], "codes of x"), (xe, xq and xq[1], "exponents of x"), (yc, yq and yq[0], "codes of y"),
                          (ye, yq and yq[1], "exponents of y")):
        if keep:
            g.check(want, what)


@pytest.mark.parametrize("rows,cols", ROWS)
@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("relu,bits", [(False, 32), (True, 32), (True, 8)])
@pytest.mark.parametrize("sums", [0, 2, 3])
def test_layer_norm_backward(rows, cols, dtype, relu, bits, sums):
    be, lib = kernels.backend(), L.lib()
    x, dy, w = make(rows, cols, dtype), make(rows, cols, dtype, 1), make(1, cols, F32, 2)[0]
    _, stats, q, _ = be.layer_norm_forward(x, w, None, 1e-5, None, relu, True, bits == 8)
    if bits == 8:
        x = None
    dx, want = be.layer_norm_backward(dy, x, q, w, stats, relu, sums)
    n = lib.dun_layer_norm_backward_workspace_floats(rows, cols, L.ROW_DTYPES[dtype], sums)
    gx, gs, gw = Guarded(rows, cols, dtype, ld=cols + 5), Guarded(max(sums, 1), cols, F32), Guarded(1 if n else 0, n, F32)
    codes, exps = (None, None) if q is None else (q[0].data_ptr(), q[1].data_ptr())
    ran(lib.dun_layer_norm_backward(
        dy.data_ptr(), cols, None if x is None else x.data_ptr(), cols, codes, exps, w.data_ptr(), stats.data_ptr(), gx.p, gx.ld,
        gs.p if sums else None, sums, gw.p if n else None, n, rows, cols, L.ROW_DTYPES[dtype], relu, stream()), "backward")
    gx.check(dx, "dx")
    gw.check(None, "workspace")
    if sums:
        gs.check(want, "sums")


@pytest.mark.parametrize("rows,cols", ROWS)
@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("relu", [False, True])
def test_pack_and_unpack(rows, cols, dtype, relu):
    be, lib = kernels.backend(), L.lib()
    x = make(rows, cols, dtype)
    q = be.act8_pack(x, relu)
    c, e = checkpoint(rows, cols)
    ran(lib.dun_act8_pack(x.data_ptr(), cols, c.p, e.p, rows, cols, L.ROW_DTYPES[dtype], relu, stream()), "pack")
    c.check(q[0], "codes")
    e.check(q[1], "exponents")
    out = Guarded(rows, cols, dtype, ld=cols + 3)
    ran(lib.dun_act8_unpack(c.p, e.p, out.p, out.ld, rows, cols, L.ROW_DTYPES[dtype], relu, stream()), "unpack")
    out.check(be.act8_unpack(q, cols, relu, dtype), "values")
    c.check(q[0], "codes")
    e.check(q[1], "exponents")


# narrow (16, 32 outputs), 64 x 64, 64 x 256, 128 x 128, 256 x 256 outputs; one range of rows and several
GRADS = [(1, 1, 1), (40, 3, 33), (3000, 1, 517), (5000, 16, 300), (600, 31, 33), (5000, 32, 1031), (33, 33, 33), (3000, 65, 517), (512, 100, 100),
         (31, 130, 70), (34, 1857, 2295), (4845, 67, 2131), (644, 1487, 2589), (7803, 1477, 69), (68, 2257, 3825), (2000, 2047, 2049)]


@pytest.mark.parametrize("rows,outs,cols", GRADS)
@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("relu", [False, True])
def test_weight_grad(rows, outs, cols, dtype, relu):
    be, lib = kernels.backend(), L.lib()
    q = be.act8_pack(make(rows, cols, F32), relu)
    c, e = checkpoint(rows, cols)
    c.view.copy_(q[0])
    e.view.copy_(q[1])
    dy = make(rows, outs, dtype, 1)
    n = lib.dun_act8_weight_grad_workspace_floats(rows, outs, cols, L.ROW_DTYPES[dtype])
    for bias in (True, False):
        dw, db = be.act8_weight_grad(dy, q, cols, relu, bias)
        gw, gb, ws = Guarded(outs, cols, F32), Guarded(1, outs, F32), Guarded(1 if n else 0, n, F32)
        ran(lib.dun_act8_weight_grad(dy.data_ptr(), outs, c.p, e.p, gw.p, gb.p if bias else None, ws.p if n else None, n, rows, outs, cols,
                                     L.ROW_DTYPES[dtype], relu, stream()), "weight_grad")
        gw.check(dw, "dw")
        gb.check(db if bias else None, "db")
        ws.check(None, "workspace")
    c.check(q[0], "codes")
    e.check(q[1], "exponents")


def test_shapes_with_and_without_a_workspace():
    """(the shapes above reach both: one workgroup or one range of rows, and several)"""
    lib = L.lib()
    norm = {lib.dun_layer_norm_backward_workspace_floats(r, c, 0, 2) > 0 for r, c in ROWS}
    grad = {lib.dun_act8_weight_grad_workspace_floats(r, o, c, 0) > 0 for r, o, c in GRADS}
    assert norm == grad == {True, False}


def test_no_rows_touch_only_the_sums():
    lib = L.lib()
    for sums in (2, 3):
        gs = Guarded(sums, 33, F32)
        ran(lib.dun_layer_norm_backward(None, 33, None, 33, None, None, None, None, None, 33, gs.p, sums, None, 0, 0, 33, 0, 0, stream()), "backward")
        gs.check(torch.zeros(sums, 33, device="cuda"), "sums")
    gw, gb = Guarded(5, 33, F32), Guarded(1, 5, F32)
    ran(lib.dun_act8_weight_grad(None, 5, None, None, gw.p, gb.p, None, 0, 0, 5, 33, 0, 0, stream()), "weight_grad")
    gw.check(torch.zeros(5, 33, device="cuda"), "dw")
    gb.check(torch.zeros(1, 5, device="cuda"), "db")
