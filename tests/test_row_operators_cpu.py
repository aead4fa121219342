"""Refusals of dun_amd.layer_norm and dun_amd.act8: nothing is launched, so no GPU is needed; and the oracle's own definitions."""
import ctypes as C

import pytest
import torch

from dun_amd import _lib, act8
from dun_amd.layer_norm import LayerNorm, Saved, layer_norm, layer_norm_backward, layer_norm_forward
from tests.row_oracle import codes_of, values_of


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 8)
    for call in (lambda: layer_norm(x), lambda: layer_norm(x.requires_grad_()), lambda: layer_norm_forward(x), lambda: act8.pack(x),
                 lambda: act8.linear(x, torch.randn(3, 8))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


@pytest.mark.parametrize("kw", [dict(weight=torch.ones(7)), dict(bias=torch.ones(9)), dict(weight=torch.ones(1, 8)),
                                dict(weight=torch.ones(8, dtype=torch.float64)), dict(residual=torch.randn(4, 7)),
                                dict(residual=torch.randn(4, 8, dtype=torch.float64)), dict(residual=torch.randn(8)),
                                dict(bits=4), dict(bits=16), dict(eps=-1e-5), dict(eps=float("nan"))])
def test_layer_norm_refuses(kw):
    x = torch.randn(4, 8)
    for fn in (layer_norm, layer_norm_forward):
        with pytest.raises(RuntimeError, match="layer_norm"):
            fn(x, **kw)


@pytest.mark.parametrize("x", [torch.randn(4, 8, dtype=torch.float64), torch.ones(4, 8, dtype=torch.int32), torch.tensor(1.0),
                               torch.empty(4, 0)])
def test_types_and_shapes_are_refused(x):
    for fn in (layer_norm, layer_norm_forward, act8.pack):
        with pytest.raises(RuntimeError):
            fn(x)


def test_backward_refuses_what_does_not_belong():
    s = Saved()
    s.shape, s.dtype, s.stats = torch.Size((4, 8)), torch.float32, torch.empty(2, 4)
    for dy in (torch.randn(4, 7), torch.randn(32), torch.randn(4, 8).bfloat16()):
        with pytest.raises(RuntimeError, match="does not go with"):
            layer_norm_backward(dy, s)


def test_checkpoints_refuse_what_does_not_belong():
    codes, exps = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8)
    p = act8.Packed8(codes, exps, (2, 2, 9), False, torch.float32)
    for args in ((codes, exps, (4, 33)), (codes, exps, (5, 9)), (codes[:, :9], exps, (4, 9)), (codes.int(), exps, (4, 9)), (codes, exps[:3], (4, 9))):
        with pytest.raises(RuntimeError, match="not a checkpoint"):
            act8.Packed8(*args, False, torch.float32)
    with pytest.raises(RuntimeError, match="unpacks to"):
        p.unpack(torch.float64)
    for dy in (torch.randn(4, 3), torch.randn(2, 3, 3), torch.randn(3, 2, 3)):
        with pytest.raises(RuntimeError, match="does not belong"):
            act8.weight_grad(dy, p)
    with pytest.raises(RuntimeError, match="float32, bfloat16"):
        act8.weight_grad(torch.randn(2, 2, 3, dtype=torch.float64), p)
    with pytest.raises(RuntimeError, match="Packed8"):
        act8.weight_grad(torch.randn(2, 2, 3), (codes, exps))


def test_linear_refuses():
    x, w = torch.randn(4, 8), torch.randn(3, 8)
    for args in ((x, w.t()), (x, torch.randn(3)), (x, w, torch.randn(4)), (x.double(), w), (x, w.bfloat16()), (x, w, torch.randn(3).double()),
                 (x, w, None, object())):
        with pytest.raises(RuntimeError, match="linear"):
            act8.linear(*args)


def test_modules_refuse():
    with pytest.raises(RuntimeError, match="last dimension"):
        LayerNorm((4, 8))
    with pytest.raises(RuntimeError, match="bits"):
        LayerNorm(8, bits=2)
    with pytest.raises(RuntimeError, match="got x"):
        LayerNorm(8)(torch.randn(4, 1))


def test_c_entries_refuse_without_launching():
    lib = _lib.lib()
    p = 1 << 20  # an address that nothing may touch
    bad = _lib.DUN_OK + 1
    fwd = lambda **k: lib.dun_layer_norm_forward(*[dict(dict(x=p, ldx=8, res=None, ldr=0, w=None, b=None, y=p, ldy=8, st=p, xc=None, xe=None,
                                                            yc=None, ye=None, rows=4, cols=8, dt=0, eps=1e-5, relu=0, s=None), **k)[n]
                                                   for n in "x ldx res ldr w b y ldy st xc xe yc ye rows cols dt eps relu s".split()])
    for k in (dict(x=None), dict(y=None), dict(ldx=7), dict(ldy=7), dict(res=p, ldr=7), dict(cols=0), dict(rows=-1), dict(dt=3), dict(xc=p),
              dict(ye=p), dict(xc=p + 4, xe=p), dict(cols=2 ** 31 - 1, ldx=2 ** 31, ldy=2 ** 31)):
        assert fwd(**k) == bad, k
        assert b"dun_layer_norm_forward" in lib.dun_last_error()
    assert fwd(rows=0, x=None) == 0
    names = "dy lddy x ldx xc xe w st dx lddx so n ws nws rows cols dt relu s".split()
    base = dict(dy=p, lddy=8, x=p, ldx=8, xc=None, xe=None, w=None, st=p, dx=p, lddx=8, so=p, n=2, ws=None, nws=0, rows=4, cols=8, dt=0, relu=0, s=None)
    for k in (dict(dy=None), dict(dx=None), dict(st=None), dict(x=None), dict(xc=p, xe=p), dict(x=None, xc=p), dict(n=1), dict(n=4), dict(so=None),
              dict(lddy=7), dict(lddx=7), dict(ldx=7), dict(dt=-1), dict(cols=0), dict(rows=5000), dict(rows=5000, ws=p, nws=10)):
        assert lib.dun_layer_norm_backward(*[dict(base, **k)[n] for n in names]) == bad, k
        assert b"dun_layer_norm_backward" in lib.dun_last_error()
    for k in (dict(x=None), dict(c=None), dict(e=None), dict(ld=7), dict(cols=0), dict(rows=-2), dict(dt=9), dict(c=p + 2)):
        a = dict(dict(x=p, ld=8, c=p, e=p, rows=4, cols=8, dt=0, relu=0, s=None), **k)
        assert lib.dun_act8_pack(*[a[n] for n in "x ld c e rows cols dt relu s".split()]) == bad, k
        assert lib.dun_act8_unpack(*[a[n] for n in "c e x ld rows cols dt relu s".split()]) == bad, k
    base = dict(dy=p, ld=6, c=p, e=p, dw=p, db=None, ws=None, nws=0, rows=4, outs=6, cols=8, dt=0, relu=0, s=None)
    for k in (dict(dy=None), dict(c=None), dict(e=None), dict(dw=None), dict(ld=5), dict(outs=0), dict(cols=0), dict(rows=-1), dict(dt=5),
              dict(c=p + 1), dict(rows=1 << 20), dict(ld=(1 << 24) + 1), dict(cols=(1 << 24) + 1)):
        assert lib.dun_act8_weight_grad(*[dict(base, **k)[n] for n in base]) == bad, k
        assert b"dun_act8_weight_grad" in lib.dun_last_error()


def test_workspaces_are_sized_for_every_shape():
    lib = _lib.lib()
    for dt in (0, 1, 2):
        assert lib.dun_layer_norm_backward_workspace_floats(0, 8, dt, 2) == 0 and lib.dun_layer_norm_backward_workspace_floats(5000, 8, dt, 0) == 0
        assert lib.dun_layer_norm_backward_workspace_floats(65536, 2048, dt, 3) % (3 * 2048) == 0
        assert lib.dun_act8_weight_grad_workspace_floats(0, 8, 8, dt) == 0
        n = lib.dun_act8_weight_grad_workspace_floats(1 << 20, 10, 100, dt)
        assert n > 0 and n % (10 * 101) == 0


def test_the_oracle_rounds_to_nearest_even_and_keeps_the_mask():
    x = torch.zeros(1, 32)
    x[0, :6] = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -126.5])
    assert values_of(x, False)[0, :6].tolist() == [127.0, 0.0, 2.0, 2.0, 0.0, -126.0]
    x[0, 0] = 127.5  # rounds to 128: the scale doubles
    q, e = codes_of(x, False)
    assert e[0, 0] == 1 and q[0, 0, 0] == 64
    x = torch.zeros(1, 32)
    x[0, :4] = torch.tensor([255.25, 1e-6, -3.0, 0.0])
    assert values_of(x, True)[0, :4].tolist() == [255.0, 1.0, 0.0, 0.0]
