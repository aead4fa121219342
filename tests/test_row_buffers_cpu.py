"""The buffers that the row operators hand to the library, on the CPU: a stand-in for the library's entries checks that every pointer it
gets lies in a tensor of the type that the kernels read or write there, with as many bytes behind it as they touch."""
import pytest
import torch

from dun_amd import _lib as L
from dun_amd import act8, kernels
from dun_amd.layer_norm import layer_norm_backward, layer_norm_forward

F32, U8 = torch.float32, torch.uint8
ROWS = {v: k for k, v in L.ROW_DTYPES.items()}


def span(rows, cols, ld):
    """Elements that rows of `cols` elements, `ld` apart, reach over."""
    return (rows - 1) * ld + cols if rows else 0


class Entries(object):
    """Stands for the library.  `seen`: every tensor that torch.empty or new_empty made or a test registered, by its address."""

    def __init__(self):
        self.real, self.seen, self.calls = L.lib(), {}, []
        for name in ("dun_layer_norm_backward_workspace_floats", "dun_act8_weight_grad_workspace_floats"):
            setattr(self, name, getattr(self.real, name))

    def hold(self, *tensors):
        for t in tensors:
            self.seen[t.data_ptr()] = t

    def need(self, p, dtype, n, what):
        t = self.seen[p]
        assert t.dtype == dtype, "%s is %s, the kernels take %s" % (what, t.dtype, dtype)
        held = t.untyped_storage().nbytes() - t.storage_offset() * t.element_size()
        assert held >= n * dtype.itemsize, "%s holds %d bytes, the kernels touch %d" % (what, held, n * dtype.itemsize)

    def codes(self, c, e, rows, cols, what):
        groups = (cols + 31) // 32
        self.need(c, U8, rows * groups * 32, what + " codes")
        self.need(e, U8, rows * groups, what + " exps")

    def dun_layer_norm_forward(self, x, ldx, res, ldr, w, b, y, ldy, stats, xc, xe, yc, ye, rows, cols, dt, eps, relu, stream):
        self.calls.append("forward")
        self.need(x, ROWS[dt], span(rows, cols, ldx), "x")
        self.need(y, ROWS[dt], span(rows, cols, ldy), "y")
        if res:
            self.need(res, ROWS[dt], span(rows, cols, ldr), "res")
        for p, n, what in ((w, cols, "w"), (b, cols, "b"), (stats, 2 * rows, "stats")):
            if p:
                self.need(p, F32, n, what)
        for c, e, what in ((xc, xe, "x"), (yc, ye, "y")):
            if c:
                self.codes(c, e, rows, cols, what)
        return 0

    def dun_layer_norm_backward(self, dy, lddy, x, ldx, xc, xe, w, stats, dx, lddx, out, sums, ws, n_ws, rows, cols, dt, relu, stream):
        self.calls.append("backward")
        self.need(dy, ROWS[dt], span(rows, cols, lddy), "dy")
        self.need(dx, ROWS[dt], span(rows, cols, lddx), "dx")
        if x:
            self.need(x, ROWS[dt], span(rows, cols, ldx), "x")
        else:
            self.codes(xc, xe, rows, cols, "x")
        if w:
            self.need(w, F32, cols, "w")
        self.need(stats, F32, 2 * rows, "stats")
        if sums:
            self.need(out, F32, sums * cols, "sums")
        need = self.dun_layer_norm_backward_workspace_floats(rows, cols, dt, sums)
        assert n_ws >= need
        if need:
            self.need(ws, F32, need, "workspace")
        return 0

    def dun_act8_pack(self, x, ldx, c, e, rows, cols, dt, relu, stream):
        self.calls.append("pack")
        self.need(x, ROWS[dt], span(rows, cols, ldx), "x")
        self.codes(c, e, rows, cols, "x")
        return 0

    def dun_act8_unpack(self, c, e, out, ldo, rows, cols, dt, relu, stream):
        self.calls.append("unpack")
        self.need(out, ROWS[dt], span(rows, cols, ldo), "out")
        self.codes(c, e, rows, cols, "x")
        return 0

    def dun_act8_weight_grad(self, dy, lddy, c, e, dw, db, ws, n_ws, rows, outs, cols, dt, relu, stream):
        self.calls.append("weight_grad")
        self.need(dy, ROWS[dt], span(rows, outs, lddy), "dy")
        self.codes(c, e, rows, cols, "x")
        self.need(dw, F32, outs * cols, "dw")
        if db:
            self.need(db, F32, outs, "db")
        need = self.dun_act8_weight_grad_workspace_floats(rows, outs, cols, dt)
        assert n_ws >= need
        if need:
            self.need(ws, F32, need, "workspace")
        return 0


@pytest.fixture
def entries(monkeypatch):
    e = Entries()
    def recorded(make):
        def made(*args, **kw):
            t = make(*args, **kw)
            e.hold(t)
            return t
        return made

    monkeypatch.setattr(torch, "empty", recorded(torch.empty))
    monkeypatch.setattr(torch.Tensor, "new_empty", recorded(torch.Tensor.new_empty))
    monkeypatch.setattr(L, "lib", lambda: e)
    monkeypatch.setattr(L, "gpu_index", lambda t: 0)
    monkeypatch.setattr(L, "elsewhere", lambda i: None)
    monkeypatch.setattr(L, "raw_stream", lambda i: 0)
    monkeypatch.setattr(L, "ptr", lambda t: None if t is None else t.data_ptr())
    monkeypatch.setattr(kernels, "_backend", None)
    yield e
    torch.set_default_dtype(torch.float32)


@pytest.mark.parametrize("default", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(4, 8), (3000, 100), (700, 1031)])
def test_buffers_whatever_the_default_type(entries, default, kind, rows, cols):
    x, res, dy = (torch.zeros(rows, cols, dtype=kind) for _ in range(3))
    w, b = torch.ones(cols), torch.zeros(cols)
    g = torch.zeros(rows, 40, dtype=kind)
    entries.hold(x, res, dy, w, b, g)
    torch.set_default_dtype(default)
    for bits in (None, 8):
        y, saved, packed = layer_norm_forward(x, w, b, residual=res, relu=True, bits=bits, pack_output=True)
        assert y.dtype == kind and saved.stats.dtype == F32
        for sum_dx, grads in ((False, True), (True, True), (False, False)):
            out = layer_norm_backward(dy, saved, sum_dx, grads)
            assert out[0].dtype == kind and all(t is None or t.dtype == F32 for t in out[1:])
    dw, db = act8.weight_grad(g, packed)
    assert dw.dtype == db.dtype == F32
    assert act8.weight_grad(g, packed, bias=False)[0].dtype == F32
    assert act8.pack(x).unpack().dtype == F32 and packed.unpack(torch.bfloat16).dtype == torch.bfloat16
    assert set(entries.calls) == {"forward", "backward", "pack", "unpack", "weight_grad"}


def test_supplied_buffers_of_another_type_are_refused(entries):
    be = kernels.backend()
    x, dy, w = torch.zeros(5000, 8), torch.zeros(5000, 8), torch.ones(8)
    entries.hold(x, dy, w)
    half = lambda *shape: torch.empty(shape, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="float32"):
        be.layer_norm_forward(x, w, None, 1e-5, stats=half(2, 5000))
    stats = be.layer_norm_forward(x, w, None, 1e-5)[1]
    with pytest.raises(RuntimeError, match="float32"):
        be.layer_norm_backward(dy, x, None, w, half(2, 5000))
    with pytest.raises(RuntimeError, match="float32"):
        be.layer_norm_backward(dy, x, None, w, stats, sums_out=half(2, 8))
    packed = be.act8_pack(x, False)
    for kw in (dict(dw=half(8, 8)), dict(db=half(8))):
        with pytest.raises(RuntimeError, match="float32"):
            be.act8_weight_grad(dy, packed, 8, False, **kw)


def test_weight_gradients_are_none_where_they_are_not_asked_for(entries):
    x = torch.zeros(6, 40)
    entries.hold(x)
    _, saved = layer_norm_forward(x)
    assert layer_norm_backward(x, saved, weight_grads=False)[1:] == (None, None)
    dx, dw, db, ds = layer_norm_backward(x, saved, sum_dx=True, weight_grads=False)
    assert dw is None and db is None and ds.shape == (40,)
    assert all(t is not None for t in layer_norm_backward(x, saved, sum_dx=True))
