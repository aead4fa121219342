"""8-bit activation checkpoints and the gradients that are taken from them.

A training step keeps every layer's input for its backward.  ``pack`` keeps it in 33 bytes per 32 consecutive columns of a row, 8-bit
codes and one power-of-two scale (1 + 1/32 bytes an element; a row's last group counts whole: 132 bytes for 100 columns, 33 for one),

    value = code * 2^e,   e the smallest integer (not below -126) for which the group's largest magnitude rounds to at
                          most 127 (255 for a rectified input, ``relu=True``: unsigned codes of max(x, 0)),

rounded to nearest even.  A positive element of a rectified input keeps a code of at least 1: ``value > 0`` is ReLU's mask.  So an element is off
by at most half a step, and a positive rectified one below half a step by less than a step; a step is at most the group's largest
magnitude / 63.75 (127.75 rectified), or 2^-126 where that is more.
A group that holds an infinity or a NaN, or whose largest magnitude would round to 2^128, reads back as NaN.

``weight_grad`` takes a Linear layer's weight gradient straight from the codes: a value is a bf16 number, an fp32
gradient the exact sum of three, so the product runs on the bf16 matrix cores without losing a bit of its operands.
``linear`` / ``Linear`` is the layer whose backward does so (float32, the framework's own products either way).

``pack``, ``unpack`` and ``weight_grad`` are not recorded by autograd; ``linear`` is differentiable (once, backward() only).  Tensors with a
forward-mode derivative are refused, and so is recording by torch.jit.trace or make_fx, which would miss the kernels.

No counterpart in the reference, which keeps everything in float32.
"""
import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import kernels


def _as_rows(t, what):
    """[..., cols] as a 2-D tensor of rows."""
    if not isinstance(t, torch.Tensor):
        raise RuntimeError("%s must be a tensor (got %s)" % (what, type(t).__name__))
    if t.dtype not in L.ROW_DTYPES:
        raise RuntimeError("%s must be float32, bfloat16 or float16 (got %s)" % (what, t.dtype))
    if t.dim() != 2:
        if t.dim() < 1:
            raise RuntimeError("%s must be a tensor of at least one dimension" % what)
        if t.shape[-1]:
            t = t.reshape(-1, t.shape[-1])
    cols = t.shape[-1]
    if not 0 < cols <= L.ROW_MOST:
        if cols == 0:
            raise RuntimeError("%s has rows of no elements: %s" % (what, tuple(t.shape)))
        raise RuntimeError("%s has more than %d elements a row: %s" % (what, L.ROW_MOST, tuple(t.shape)))
    return t


class Packed8(object):
    """An 8-bit checkpoint of a tensor: ``codes`` uint8 [rows, 32 G] (signed codes are stored + 128) and ``exps`` uint8
    [rows, G] (exponents + 127), G = ceil(cols / 32)."""
    __slots__ = ("codes", "exps", "shape", "relu", "dtype")

    def __init__(self, codes, exps, shape, relu, dtype):
        self.codes, self.exps, self.shape, self.relu, self.dtype = codes, exps, tuple(shape), bool(relu), dtype
        cols = self.shape[-1]
        groups = (cols + L.ACT8_GROUP - 1) // L.ACT8_GROUP
        rows = 1
        for n in self.shape[:-1]:
            rows *= n
        for t, want in ((codes, (rows, groups * L.ACT8_GROUP)), (exps, (rows, groups))):
            if t.dtype != torch.uint8 or tuple(t.shape) != want or not t.is_contiguous() or t.device != codes.device:
                raise RuntimeError("not a checkpoint of a tensor of shape %s: uint8 %s wanted, got %s %s"
                                   % (self.shape, want, t.dtype, tuple(t.shape)))

    @classmethod
    def _of(cls, packed, shape, relu, dtype):
        """Around buffers that were made for it (nothing to check)."""
        p = object.__new__(cls)
        p.codes, p.exps = packed
        p.shape, p.relu, p.dtype = tuple(shape), relu, dtype
        return p

    @property
    def packed(self):
        return self.codes, self.exps

    @property
    def nbytes(self):
        return self.codes.numel() + self.exps.numel()

    def unpack(self, dtype=torch.float32):
        """The values that the codes stand for (exact in float32 and bfloat16)."""
        if dtype not in L.ROW_DTYPES:
            raise RuntimeError("a checkpoint unpacks to float32, bfloat16 or float16 (got %s)" % dtype)
        v = kernels.backend().act8_unpack((self.codes, self.exps), self.shape[-1], self.relu, dtype)
        return v if len(self.shape) == 2 else v.view(self.shape)


def pack(x, relu=False):
    """The 8-bit checkpoint of ``x`` [..., cols], or of max(x, 0) with ``relu``."""
    relu = bool(relu)
    if forward_ad._current_level >= 0:
        L.no_tangents("pack", x)
    return Packed8._of(kernels.backend().act8_pack(_as_rows(x, "pack: x"), relu), x.shape, relu, x.dtype)


def weight_grad(dy, packed, bias=True):
    """(dw [outs, cols], db [outs]): the float32 gradients of the weight and bias of a Linear layer, from the gradient
    ``dy`` [..., outs] of its output and the checkpoint of its input.  ``bias=False``: db is None.  An infinity in a float32 or
    float16 ``dy`` counts as NaN for its output's weights (its parts are infinity and NaN)."""
    if not isinstance(packed, Packed8):
        raise RuntimeError("weight_grad: packed must be a Packed8 (got %s)" % type(packed).__name__)
    dy2 = _as_rows(dy, "weight_grad: dy")
    if forward_ad._current_level >= 0:
        L.no_tangents("weight_grad", dy)
    if dy.shape[:-1] != packed.shape[:-1] or dy.get_device() != packed.codes.get_device():
        raise RuntimeError("weight_grad: dy %s on %s does not belong to a checkpoint of %s on %s"
                           % (tuple(dy.shape), dy.device, packed.shape, packed.codes.device))
    return kernels.backend().act8_weight_grad(dy2, (packed.codes, packed.exps), packed.shape[-1], packed.relu, bool(bias))


class _Linear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, packed, keep):
        be = kernels.backend()
        x2 = x.detach().reshape(-1, x.shape[-1]).contiguous()
        w = weight.detach().contiguous()
        rows, cols, outs = x2.shape[0], x2.shape[1], w.shape[0]
        ctx.shape, ctx.has_bias, ctx.relu = tuple(x.shape), bias is not None, False
        codes = exps = None
        if keep:
            codes, exps = be.act8_pack(x2, False) if packed is None else packed.packed
            ctx.relu = False if packed is None else packed.relu
        ctx.save_for_backward(weight, codes, exps)
        if rows == 0:
            return x.new_empty(x.shape[:-1] + (outs,))
        with torch.cuda.device(L.gpu_index(x2)):
            y = be.gemm(x2, w, rows, outs, cols, bias=None if bias is None else bias.detach().contiguous())
        return y.view(x.shape[:-1] + (outs,))

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        be = kernels.backend()
        weight, codes, exps = ctx.saved_tensors
        outs, cols = weight.shape
        dy2 = dy.reshape(-1, outs).contiguous()
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            if dy2.shape[0] == 0:
                dx = dy.new_empty(ctx.shape)
            else:
                with torch.cuda.device(L.gpu_index(dy2)):
                    dx = be.gemm(dy2, weight.detach().contiguous(), dy2.shape[0], cols, outs, b_kcontig=False).view(ctx.shape)
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
            dw, db = be.act8_weight_grad(dy2, (codes, exps), cols, ctx.relu, want_bias=ctx.has_bias)
        return dx, dw if ctx.needs_input_grad[1] else None, db if ctx.needs_input_grad[2] else None, None, None


def linear(x, weight, bias=None, packed=None):
    """x weight^T + bias, like torch.nn.functional.linear, keeping ``x`` for the backward in 8 bits.  ``packed``: the
    checkpoint of ``x`` where the caller has it already (layer_norm's ``pack_output``; a rectified checkpoint belongs to a
    rectified x).  float32."""
    for t, what in ((x, "x"), (weight, "weight"), (bias, "bias")):
        if t is not None and (t.dtype != torch.float32 or t.device != x.device):
            raise RuntimeError("linear: %s must be float32 on %s (got %s on %s)" % (what, x.device, t.dtype, t.device))
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or weight.numel() == 0:
        raise RuntimeError("linear: x %s does not go with weight %s" % (tuple(x.shape), tuple(weight.shape)))
    if x.numel() // x.shape[-1] >= 1 << 31 or max(weight.shape) >= 1 << 31:
        raise RuntimeError("linear: x %s and weight %s: at most 2^31 - 1 rows, inputs and outputs" % (tuple(x.shape), tuple(weight.shape)))
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise RuntimeError("linear: bias %s does not go with weight %s" % (tuple(bias.shape), tuple(weight.shape)))
    if packed is not None and (not isinstance(packed, Packed8) or packed.shape != tuple(x.shape) or packed.codes.device != x.device):
        raise RuntimeError("linear: packed is not a checkpoint of x %s" % (tuple(x.shape),))
    if forward_ad._current_level >= 0:
        L.no_tangents("linear", x, weight, bias)
    # (needs_input_grad does not know of no_grad: a prediction would pack what nothing reads)
    keep = torch.is_grad_enabled() and (weight.requires_grad or (bias is not None and bias.requires_grad))
    return _Linear8.apply(x, weight, bias, packed, keep)


class Linear(nn.Linear):
    """nn.Linear that keeps its input for the backward in 8 bits; same parameters and state_dict."""

    def forward(self, x, packed=None):
        return linear(x, self.weight, self.bias, packed)
