"""Row operators under forward-mode differentiation and under recorders of torch operators: a result without its tangent, or a recording
without the kernels, would be silently wrong, so both are refused.  On the CPU a stand-in takes the place of the library's entries."""
import contextlib

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from dun_amd import _lib as L
from dun_amd import act8, kernels
from dun_amd.layer_norm import LayerNorm, layer_norm, layer_norm_backward, layer_norm_forward
from tests.test_row_buffers_cpu import Entries

pytestmark = pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
DEVICES = [pytest.param("cpu", id="cpu"), pytest.param("cuda", marks=pytest.mark.gpu, id="gpu")]


@pytest.fixture(params=DEVICES)
def dev(request, monkeypatch):
    if request.param == "cpu":
        e = Entries()
        e.need = lambda *args: None
        index = L.gpu_index

        class OnGpu(object):
            get_device = staticmethod(lambda: 0)

        monkeypatch.setattr(L, "lib", lambda: e)
        monkeypatch.setattr(L, "gpu_index", lambda t: index(OnGpu()))
        monkeypatch.setattr(L, "elsewhere", lambda i: None)
        monkeypatch.setattr(L, "raw_stream", lambda i: 0)
        monkeypatch.setattr(L, "ptr", lambda t: None if t is None else t.data_ptr())
        monkeypatch.setattr(torch.cuda, "device", lambda i: contextlib.nullcontext())
        monkeypatch.setattr(kernels, "_backend", None)
        monkeypatch.setattr(kernels.HipBackend, "gemm", lambda self, A, B, M, N, K, **kw: A.new_zeros(M, N))
    return request.param


def calls(dev):
    """{name: (function of one tensor, that tensor)}: every operator, differentiated by every input that has a derivative"""
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to(dev)
    x, res, w, b, W, c, dy = r(6, 40), r(6, 40), r(40), r(40), r(5, 40), r(5), r(6, 5)
    packed = act8.pack(x)
    saved = layer_norm_forward(x, w, b)[1]
    norm = LayerNorm(40).to(dev)
    for p in norm.parameters():
        p.requires_grad_(False)
    return {
        "x": (lambda t: layer_norm(t, w, b, residual=res), x), "weight": (lambda t: layer_norm(x, t, b), w),
        "bias": (lambda t: layer_norm(x, w, t), b), "residual": (lambda t: layer_norm(x, w, b, residual=t), res),
        "packed output": (lambda t: layer_norm(t, w, b, bits=8, pack_output=True)[0], x), "module": (norm, x),
        "forward half": (lambda t: layer_norm_forward(t, w, b)[0], x), "backward half": (lambda t: layer_norm_backward(t, saved)[0], r(6, 40)),
        "pack": (lambda t: act8.pack(t).codes, x), "unpack": (lambda t: act8.pack(t).unpack(), x),
        "weight_grad": (lambda t: act8.weight_grad(t, packed)[0], dy), "linear x": (lambda t: act8.linear(t, W, c), x),
        "linear weight": (lambda t: act8.linear(x, t, c), W), "linear bias": (lambda t: act8.linear(x, W, t), c)}


NAMES = ["x", "weight", "bias", "residual", "packed output", "module", "forward half", "backward half", "pack", "unpack", "weight_grad",
         "linear x", "linear weight", "linear bias"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(dev, name, grad):
    f, t = calls(dev)[name]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        f(t)  # (no tangent, nothing to lose)
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(forward_ad.make_dual(t, torch.ones_like(t)))
        if grad and name not in ("forward half", "backward half", "pack", "unpack", "weight_grad"):
            with pytest.raises(RuntimeError, match="forward|jvp"):
                f(forward_ad.make_dual(t.clone().requires_grad_(), torch.ones_like(t)))
    with pytest.raises(RuntimeError):
        torch.func.jvp(f, (t,), (torch.ones_like(t),))


@pytest.mark.parametrize("name", NAMES)
def test_recorders_are_refused(dev, name):
    f, t = calls(dev)[name]
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="recorded graph"):
            torch.jit.trace(f, (t,), check_trace=False)
    with pytest.raises(RuntimeError, match="recorded graph"):
        torch.jit.trace(f, (t.clone().requires_grad_(),), check_trace=False)
    with pytest.raises(RuntimeError, match="recorded graph"):
        make_fx(f, tracing_mode="real")(t)
    f(t)  # (and nothing of it stays)


def test_other_modes_of_dispatch_are_no_recording(dev):
    from torch.utils.flop_counter import FlopCounterMode
    f, t = calls(dev)["x"]
    want = f(t)
    with FlopCounterMode(display=False):
        got = f(t)
    assert dev == "cpu" or torch.equal(got, want)


@pytest.mark.gpu
def test_a_trunk_is_not_recorded():
    from tests.test_ln_trunk_gpu import build
    m = build(bits=8).model.eval()
    x = torch.randn(9, 13, device="cuda")
    with torch.no_grad(), pytest.raises(RuntimeError, match="recorded graph"):
        torch.jit.trace(m, (x,), check_trace=False)
    assert m(x).shape == (5, 9, 1)
