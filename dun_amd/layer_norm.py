"""Layer normalisation over the last dimension, with the pieces that a residual block puts around it.

    z = x, or max(x, 0) with ``relu``
    y = [residual +] (z - mean) * rstd * weight + bias,   rstd = 1 / sqrt(var + eps), biased variance, per row

    g = dy * weight,  xhat = (z - mean) * rstd
    dx = rstd * (g - mean(g) - xhat * mean(g * xhat))  [0 where z <= 0 with ``relu``],  dresidual = dy
    dweight = sum_rows dy * xhat,  dbias = sum_rows dy

``bits=8`` keeps z for the backward as an 8-bit checkpoint (dun_amd.act8): xhat is then taken from the checkpoint's values and the
forward's mean and rstd.  float32, bfloat16 and float16 rows; statistics and sums in float32; weight and bias of any of these types.

``layer_norm`` is differentiable (once, backward() only: tensors with a forward-mode derivative are refused, and so is recording by
torch.jit.trace or make_fx, which would miss the kernels); ``layer_norm_forward`` / ``layer_norm_backward`` are the two halves for callers
that run their backward themselves, like the trunks of this package.  Both can be captured into a HIP graph.  A captured
``backward()`` goes by torch's rule for every operator: no earlier autograd graph of the same leaves may be alive (its
gradient accumulators belong to another stream, which ends the process); the two halves have none.  Batches couple nowhere: no running statistics, no
exchange between ranks, a batch of one row trains.

The reference's blocks know BatchNorm only (src/DUN/layers.py:33-53).
"""
import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import kernels
from .act8 import Packed8, _as_rows


def _vector(t, cols, x, what):
    """weight / bias as the kernels take it: float32, contiguous."""
    if t.dim() != 1 or t.shape[0] != cols:
        raise RuntimeError("layer_norm: %s %s does not go with rows of %d elements" % (what, tuple(t.shape), cols))
    if t.get_device() != x.get_device():
        raise RuntimeError("layer_norm: %s is on %s, x on %s" % (what, t.device, x.device))
    if t.dtype is not torch.float32:
        if t.dtype not in (torch.bfloat16, torch.float16):
            raise RuntimeError("layer_norm: %s must be float32, bfloat16 or float16 (got %s)" % (what, t.dtype))
        t = t.detach().float()
    return t if t.is_contiguous() else t.detach().contiguous()


def _checked(x, weight, bias, eps, residual, bits):
    x2 = _as_rows(x, "layer_norm: x")
    if forward_ad._current_level >= 0:
        L.no_tangents("layer_norm", x, weight, bias, residual)
    cols = x2.shape[1]
    w = None if weight is None else _vector(weight, cols, x, "weight")
    b = None if bias is None else _vector(bias, cols, x, "bias")
    if not eps >= 0:
        raise RuntimeError("layer_norm: eps must not be negative (got %r)" % (eps,))
    if bits not in (None, 8, 32):
        raise RuntimeError("layer_norm: bits is 32 (or None) or 8 (got %r)" % (bits,))
    r2 = None
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.get_device() != x.get_device():
            raise RuntimeError("layer_norm: residual %s %s on %s does not go with x %s %s on %s"
                               % (tuple(residual.shape), residual.dtype, residual.device, tuple(x.shape), x.dtype, x.device))
        r2 = _as_rows(residual, "layer_norm: residual")
    return x2, w, b, r2


class Saved(object):
    """What ``layer_norm_forward`` keeps for the backward."""
    __slots__ = ("x", "packed", "w", "stats", "relu", "shape", "dtype", "w_dtype", "b_dtype")


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5, residual=None, relu=False, bits=None, pack_output=False):
    """-> (y, saved), or (y, saved, Packed8 of y) with ``pack_output``.  Not recorded by autograd; ``saved`` refers to
    ``weight`` itself and, unless ``bits`` is 8, to ``x``: they must not change before ``layer_norm_backward``."""
    x2, w, b, r2 = _checked(x, weight, bias, eps, residual, bits)
    relu = bool(relu)
    y, stats, xq, yq = kernels.backend().layer_norm_forward(x2, w, b, eps, r2, relu, True, bits == 8, bool(pack_output))
    s = Saved()
    s.x, s.packed, s.w, s.stats, s.relu = (x2.detach() if xq is None else None), xq, w, stats, relu
    s.shape, s.dtype = x.shape, x.dtype
    s.w_dtype = None if weight is None else weight.dtype
    s.b_dtype = None if bias is None else bias.dtype
    y = y if x.dim() == 2 else y.view(x.shape)
    if pack_output:
        return y, s, Packed8._of(yq, x.shape, False, x.dtype)
    return y, s


def layer_norm_backward(dy, saved, sum_dx=False, weight_grads=True):
    """-> (dx, dweight, dbias[, sum_rows dx]); the residual's gradient is ``dy``.  dweight / dbias in the types of weight and
    bias (float32 where there was none), None without ``weight_grads``; with ``sum_dx`` also the float32 bias gradient of
    the Linear that made x."""
    if dy.shape != saved.shape or dy.dtype != saved.dtype or dy.get_device() != saved.stats.get_device():
        raise RuntimeError("layer_norm_backward: dy %s %s on %s does not go with x %s %s on %s"
                           % (tuple(dy.shape), dy.dtype, dy.device, tuple(saved.shape), saved.dtype, saved.stats.device))
    if forward_ad._current_level >= 0:
        L.no_tangents("layer_norm_backward", dy)
    dy2 = dy if dy.dim() == 2 else dy.reshape(-1, dy.shape[-1])
    dx, sums = kernels.backend().layer_norm_backward(dy2, saved.x, saved.packed, saved.w, saved.stats, saved.relu,
                                                     3 if sum_dx else 2 if weight_grads else 0)
    if sums is None:
        return dx if dy.dim() == 2 else dx.view(saved.shape), None, None
    rows = sums.unbind(0)
    dw, db = (rows[0], rows[1]) if weight_grads else (None, None)
    if weight_grads and saved.w_dtype not in (None, torch.float32):
        dw = dw.to(saved.w_dtype)
    if weight_grads and saved.b_dtype not in (None, torch.float32):
        db = db.to(saved.b_dtype)
    dx = dx if dy.dim() == 2 else dx.view(saved.shape)
    return (dx, dw, db, rows[2]) if sum_dx else (dx, dw, db)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps, relu, bits, pack_output):
        out = layer_norm_forward(x, weight, bias, eps, residual, relu, bits, pack_output)
        y, s = out[0], out[1]
        codes, exps = (None, None) if s.packed is None else s.packed
        # (weight's float32 copy, if one was made, is not what autograd watches: the parameter itself is saved)
        ctx.save_for_backward(x if s.packed is None else None, codes, exps, weight, s.stats)
        ctx.info = (s.relu, s.w_dtype, s.b_dtype, x.shape, x.dtype)
        if not pack_output:
            return y
        yq = out[2]
        ctx.mark_non_differentiable(yq.codes, yq.exps)
        return y, yq.codes, yq.exps

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, *unused):
        x, codes, exps, weight, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if need[0] or need[1] or need[2]:
            s = Saved()
            s.relu, s.w_dtype, s.b_dtype, s.shape, s.dtype = ctx.info
            s.x = None if x is None else _as_rows(x.detach(), "layer_norm: x")
            s.packed = None if codes is None else (codes, exps)
            s.w = None if weight is None else _vector(weight, s.shape[-1], stats, "weight")
            s.stats = stats
            dx, dw, db = layer_norm_backward(dy, s, weight_grads=need[1] or need[2])
        return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None, dy if need[3] else None,
                None, None, None, None)


def layer_norm(x, weight=None, bias=None, eps=1e-5, residual=None, relu=False, bits=None, pack_output=False):
    """Layer norm of the rows of ``x`` [..., cols] (see the module's head).  ``pack_output``: -> (y, Packed8 of y), for
    the ``act8.linear`` that reads y next."""
    if not torch.is_grad_enabled() or not (x.requires_grad or (weight is not None and weight.requires_grad)
                                           or (bias is not None and bias.requires_grad)
                                           or (residual is not None and residual.requires_grad)):
        x2, w, b, r2 = _checked(x, weight, bias, eps, residual, bits)
        y, _, _, yq = kernels.backend().layer_norm_forward(x2, w, b, eps, r2, bool(relu), False, False, bool(pack_output))
        y = y if x.dim() == 2 else y.view(x.shape)
        return (y, Packed8._of(yq, x.shape, False, x.dtype)) if pack_output else y
    out = _LayerNorm.apply(x, weight, bias, residual, eps, relu, bits, bool(pack_output))
    if pack_output:
        return out[0], Packed8._of((out[1], out[2]), x.shape, False, x.dtype)
    return out


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm over the last dimension on the HIP kernels; same parameters and state_dict.  ``bits=8``: 8-bit
    checkpoint for the backward."""

    def __init__(self, normalized_shape, eps=1e-5, elementwise_affine=True, bias=True, device=None, dtype=None, bits=None):
        super(LayerNorm, self).__init__(normalized_shape, eps, elementwise_affine, bias, device, dtype)
        if len(self.normalized_shape) != 1:
            raise RuntimeError("LayerNorm normalises the last dimension only (got %s)" % (self.normalized_shape,))
        if bits not in (None, 8, 32):
            raise RuntimeError("LayerNorm: bits is 32 (or None) or 8 (got %r)" % (bits,))
        self.bits = bits

    def forward(self, x, residual=None, relu=False):
        if x.shape[-1] != self.normalized_shape[0]:
            raise RuntimeError("LayerNorm over %d elements got x %s" % (self.normalized_shape[0], tuple(x.shape)))
        return layer_norm(x, self.weight, self.bias, self.eps, residual, relu, self.bits)
