"""Residual-MLP / plain-MLP DUN trunks with the reference's constructor and attribute surface.

Reference: src/DUN/stochastic_fc_models.py:7-80.  ``forward(x, depth=None)`` returns ``act_vec [D,B,O]``
(the north-star's "forward_get_acts"; an alias of that name is provided).  All arithmetic of ``forward``
and its backward runs in the HIP trunk kernels (dun_amd/csrc/trunk.hip, gemm.hip, head.hip): the module's
parameters are views into one flat fp32 buffer that the kernels, the fused SGD step and the gradient
all-reduce address directly; gradients land in a second flat buffer whose views are the parameters' ``.grad``.
"""
import weakref

import torch
import torch.nn as nn

from . import kernels
from .layers import bern_LNBlock, bern_MLPBlock, bern_MLPBlock_nores

_SEG_ALIGN = 64  # floats: every segment of the flat buffers starts on a 256-byte boundary
_KINDS = ("w_in", "b_in", "w_out", "b_out", "w", "b", "gamma", "beta")


def _round_up(n, a):
    return (n + a - 1) // a * a


class _FcForward(torch.autograd.Function):
    """Autograd node of the whole trunk.  Parameter gradients are written by the kernels straight into the
    flat gradient buffer (``p.grad`` views), not returned to autograd, and overwrite what was there."""

    @staticmethod
    def forward(ctx, model, x, depth, objective, *params):
        buf = model._run_forward(x, depth, True, objective)
        ctx.model, ctx.buf, ctx.generation = model, buf, buf.generation
        # The returned tensor becomes this node's output (grad_fn -> node -> parameters -> model).  Left in the buffer
        # object it would close model -> buffers -> act -> node -> model through the C++ autograd graph, which
        # Python's collector cannot see: a dropped model kept its activation buffers (55 GB at C3) allocated.
        act, buf.act = buf.act, None
        return act

    @staticmethod
    def backward(ctx, dact):
        model, buf = ctx.model, ctx.buf
        if buf is None:
            raise RuntimeError("the trunk's backward ran already (its buffers are reused by the next forward)")
        ctx.model = ctx.buf = None  # a kept act_vec does not pin the buffers
        if buf.generation != ctx.generation:
            # H / Z / BatchNorm statistics live in ONE buffer set per (batch, depth, mode): a later train-mode forward
            # of the same batch size (also under no_grad, e.g. a sweep with train_bn=True) has overwritten what this
            # backward needs.  Gradients are also written, not accumulated (no micro-batch accumulation).
            raise RuntimeError("the trunk's activation buffers were reused by a later train-mode forward of the same batch "
                               "size before this backward ran; run backward before the next forward")
        model._run_backward(buf, dact)
        return (None, None, None, None) + (None,) * len(model._param_list)


class arq_uncert_fc_resnet(nn.Module):
    residual = True
    _block_cls = bern_MLPBlock

    def __init__(self, input_dim, output_dim, width, n_layers, w_prior=None, BMA_prior=False):
        super(arq_uncert_fc_resnet, self).__init__()
        self.input_dim = input_dim
        self.output_dim = output_dim
        # same construction order as the reference, so an identical torch seed gives identical initial weights
        self.input_layer = nn.Linear(self.input_dim, width)
        self.output_layer = nn.Linear(width, self.output_dim)
        self.n_layers = n_layers
        self.width = width
        self.w_prior = w_prior
        self.BMA_prior = BMA_prior
        if not isinstance(self.w_prior, list) and self.w_prior is not None:
            self.w_prior = [self.w_prior for _ in range(self.n_layers + 1)]
        self.stochstic_layers = nn.ModuleList()
        for _ in range(self.n_layers):
            self.stochstic_layers.append(self._block_cls(width))
        self.bn_eps, self.bn_momentum = 1e-5, 0.1
        self._dist = None      # set by dun_amd.distributed.shard(): batch-sharded data parallelism
        self._fc_cache = {}
        self._flatten()

    # ---- flat parameter / gradient storage ---------------------------------------------------------
    def _segments(self):
        W, L, O, din = self.width, self.n_layers, self.output_dim, self.input_dim
        sizes = dict(w_in=W * din, b_in=W, w_out=O * W, b_out=O, w=L * W * W, b=L * W, gamma=L * W, beta=L * W)
        shapes = dict(w_in=(W, din), b_in=(W,), w_out=(O, W), b_out=(O,), w=(L, W, W), b=(L, W), gamma=(L, W),
                      beta=(L, W))
        offs, o = {}, 0
        for k in _KINDS:
            offs[k] = o
            o += _round_up(sizes[k], _SEG_ALIGN)
        return sizes, shapes, offs, max(o, _SEG_ALIGN)

    def _module_params(self):
        """(kind, layer index or None, Parameter) in flat-buffer order."""
        out = [("w_in", None, self.input_layer.weight), ("b_in", None, self.input_layer.bias),
               ("w_out", None, self.output_layer.weight), ("b_out", None, self.output_layer.bias)]
        for kind, sub, attr in (("w", 0, "weight"), ("b", 0, "bias"), ("gamma", 2, "weight"), ("beta", 2, "bias")):
            for i, blk in enumerate(self.stochstic_layers):
                out.append((kind, i, getattr(blk.block[sub], attr)))
        return out

    def _flatten(self):
        sizes, shapes, offs, total = self._segments()
        dev = self.input_layer.weight.device
        flat = torch.zeros(total, device=dev, dtype=torch.float32)
        gflat = torch.zeros(total, device=dev, dtype=torch.float32)
        self.stacked, self.stacked_grad = {}, {}
        for k in _KINDS:
            self.stacked[k] = flat[offs[k]:offs[k] + sizes[k]].view(shapes[k])
            self.stacked_grad[k] = gflat[offs[k]:offs[k] + sizes[k]].view(shapes[k])
        self._param_list, self._grad_views = [], []
        with torch.no_grad():
            for kind, i, p in self._module_params():
                dst = self.stacked[kind] if i is None else self.stacked[kind][i]
                gdst = self.stacked_grad[kind] if i is None else self.stacked_grad[kind][i]
                dst.copy_(p.data.to(torch.float32))
                p.data = dst
                p.grad = gdst
                p._dun_flat_owner = self
                self._param_list.append(p)
                self._grad_views.append(gdst)
            rm, rv, nbt = self._flatten_norm(dev)
        self.flat_params, self.flat_grads = flat, gflat
        # captured steps hold the addresses of the buffers they were captured on: a rebuilt flat buffer (load_state_dict,
        # .to()) may land on the old parameter address while its gradient buffer does not, so the wrappers key their
        # graphs on this counter too
        self._flat_generation = self.__dict__.get("_flat_generation", 0) + 1
        self.running_mean, self.running_var, self.num_batches_tracked = rm, rv, nbt
        self._fc_cache = {}
        # every parameter of the module tree lives in the flat buffer (what the whole-step hipGraph relies on)
        self._all_params_flat = all(getattr(q, "_dun_flat_owner", None) is self for q in self.parameters())

    def _flatten_norm(self, dev):
        """BatchNorm's buffers of all blocks as rows of three tensors."""
        L, W = self.n_layers, self.width
        rm = torch.zeros(L, W, device=dev)
        rv = torch.ones(L, W, device=dev)
        nbt = torch.zeros(L, device=dev, dtype=torch.int64)
        for i, blk in enumerate(self.stochstic_layers):
            bn = blk.block[2]
            rm[i].copy_(bn.running_mean)
            rv[i].copy_(bn.running_var)
            nbt[i] = bn.num_batches_tracked
            bn.running_mean = rm[i]
            bn.running_var = rv[i]
            bn.num_batches_tracked = nbt[i]
        return rm, rv, nbt

    def _apply(self, fn, *args, **kwargs):
        super(arq_uncert_fc_resnet, self)._apply(fn, *args, **kwargs)
        if hasattr(self, "flat_params"):
            self._flatten()  # .cuda()/.to() re-created the tensors: rebuild the flat views on the new device
        return self

    def load_state_dict(self, state_dict, strict=True, **kw):
        out = super(arq_uncert_fc_resnet, self).load_state_dict(state_dict, strict=strict, **kw)
        self._flatten()
        return out

    def __getstate__(self):
        st = self.__dict__.copy()
        st["_fc_cache"] = {}
        st["_dist"] = None
        st.pop("_mode_synced", None)
        for k in ("stacked", "stacked_grad", "_param_list", "_grad_views", "flat_params", "flat_grads",
                  "running_mean", "running_var", "num_batches_tracked"):
            st.pop(k, None)
        return st

    def __setstate__(self, st):
        super(arq_uncert_fc_resnet, self).__setstate__(st)
        self._flatten()

    def train(self, mode=True):
        """nn.Module.train walks the ~30 sub-modules (tens of microseconds per call, and fit / eval / predict call it
        every step like the reference does): skipped when the tree is already in that mode.  The kernels only read
        this module's own flag; the children's flags matter to the torch cold path (vec_forward) and are kept in
        step as long as modes are switched through this module, which is what the wrappers do."""
        if self.training == mode and self.__dict__.get("_mode_synced") == mode:
            return self
        super(arq_uncert_fc_resnet, self).train(mode)
        self.__dict__["_mode_synced"] = mode
        return self

    # ---- weight priors: O(#params) torch reductions, not part of the per-sample path ----
    def apply_prior(self, module, prior_f):
        if isinstance(module, (nn.Linear, nn.Conv2d, nn.Conv1d)):
            self.loglike = self.loglike + prior_f(module.weight)
            self.loglike = self.loglike + prior_f(module.bias)

    def get_w_prior_loglike(self, k=None):
        if k is None:
            k = self.n_layers
        if self.w_prior is None:
            return self.input_layer.bias.data.new_zeros(k + 1)
        self.loglike = 0
        self.input_layer.apply(lambda m: self.apply_prior(m, self.w_prior[0]))
        self.output_layer.apply(lambda m: self.apply_prior(m, self.w_prior[0]))
        self.loglikes = [self.loglike]
        for idx, layer in enumerate(self.stochstic_layers[:k]):
            self.loglike = 0
            layer.apply(lambda m: self.apply_prior(m, self.w_prior[idx + 1]))
            self.loglikes.append(self.loglike)
        loglike_vec = torch.stack(self.loglikes, dim=0)
        if self.BMA_prior:
            loglike_vec = loglike_vec.unsqueeze(0).repeat(k + 1, 1).tril(diagonal=0).sum(dim=1)
        return loglike_vec.sum(dim=0)

    # ---- cold path: explicit 0/1 mask per block, torch ops (plots only) -------------------
    def vec_forward(self, x, vec):
        assert vec.shape[0] == self.n_layers
        x = self.input_layer(x)
        for i in range(self.n_layers):
            x = self.stochstic_layers[i](x, vec[i])
        return self.output_layer(x)

    # ---- hot path ---------------------------------------------------------------------------------------
    def _get_buffers(self, B, depth, train):
        key = (B, depth, bool(train))
        buf = self._fc_cache.get(key)
        if buf is None:
            if len(self._fc_cache) >= 4:  # keep the cache bounded: training + a few inference shapes
                for k in [k for k in self._fc_cache if not k[2]][:1] or list(self._fc_cache)[:1]:
                    del self._fc_cache[k]
            buf = self._make_buffers(B, depth, train)
            self._fc_cache[key] = buf
        return buf

    def _make_buffers(self, B, depth, train):
        return kernels.backend().fc_buffers(self, B, depth, train)

    supports_head_objective = True  # forward(x, objective=HeadObjective): likelihood pass inside the head kernels

    def _run_forward(self, x, depth, train, objective=None):
        if x.dim() != 2 or x.shape[1] != self.input_dim:
            raise RuntimeError("expected x of shape [B, %d], got %s" % (self.input_dim, tuple(x.shape)))
        if train and depth > 0:
            # nn.BatchNorm1d in training mode (torch.nn.functional.batch_norm -> _verify_batch_size): a batch of one
            # row has no variance.  The reference's blocks raise this from a ragged last batch of size 1; here the
            # unbiased running-variance update would divide by n - 1 = 0 and poison the running statistics silently.
            dist = self._dist
            n_stat = dist.global_batch(x.shape[0]) if (dist is not None and dist.sync_bn) else x.shape[0]
            if n_stat <= 1:
                raise ValueError("Expected more than 1 value per channel when training, got input size %s"
                                 % (torch.Size([x.shape[0], self.width]),))
        be = kernels.backend()
        x = x.detach().to(torch.float32).contiguous()
        buf = self._get_buffers(x.shape[0], depth, train)
        buf.generation += 1
        buf.new_act()
        buf.set_input(x)
        buf.set_objective(objective if self.output_dim == 1 else None)
        dist = self._dist
        if dist is None or not (train and dist.sync_bn) or depth == 0:
            be.fc_forward(buf)
        else:
            # Staged at the BatchNorm exchanges.  Where block_norm(i) writes act[i+1] itself (row-owned BatchNorm apply
            # + head: buf.head_fused) only depth 0 needs the head kernel; otherwise the shared head runs depth by depth
            # on the hidden state block i started from, with dist.async_forward_bn UNDER the exchange of block i
            gb = dist.global_batch(x.shape[0])
            fused = buf.head_fused
            be.fc_input_layer(buf)
            if fused:
                be.fc_head_depth(buf, 0)
            for i in range(depth):
                be.fc_block_linear(buf, i)
                if dist.async_forward_bn and not fused:
                    h = dist.all_reduce_async(buf.bn_sums)
                    be.fc_head_depth(buf, i)
                    if h is not None:
                        h.wait()
                else:
                    dist.all_reduce(buf.bn_sums)
                    if not fused:
                        be.fc_head_depth(buf, i)
                be.fc_block_norm(buf, i, gb)
            if not fused:
                be.fc_head_depth(buf, depth)
        # (nn.BatchNorm1d.num_batches_tracked of the blocks that ran is advanced by the kernels that update the running
        # statistics: dun_fc_ctx.num_batches_tracked)
        return buf

    def _run_backward(self, buf, dact):
        be = kernels.backend()
        buf.ensure_backward()
        buf.set_dact(dact.detach().to(torch.float32).contiguous())
        dist = self._dist
        if dist is None:
            be.fc_backward(buf)
        else:
            gb = dist.global_batch(buf.B)
            be.fc_bwd_begin(buf)
            # The BatchNorm exchange of block i (16 KB, latency bound) sits between its column reduction and its dU;
            # the weight-gradient GEMM of block i+1 needs neither, so it is deferred to run UNDER that exchange (dU of
            # block i+1 stays in place until bwd_block_dx(i)).  The gradient message of block i+1 follows the small
            # exchange on the single communicator stream and has a dX GEMM + a reduction + a dW GEMM of time before
            # the next small message is queued behind it.
            # Weight gradients leave in buckets of `dist.grad_bucket_blocks` consecutive blocks (one contiguous slice
            # of the stacked gradient): fewer, larger messages for the per-link-bound xGMI rings.
            deferred = None
            sent_from = self.n_layers  # blocks [sent_from, L) are on their way

            def dw_and_send(j):
                nonlocal sent_from
                be.fc_bwd_block_dw(buf, j)
                if sent_from - j >= dist.grad_bucket_blocks or j == 0:
                    dist.reduce_gradient_async(self.stacked_grad["w"][j:sent_from])
                    sent_from = j

            for i in range(self.n_layers - 1, -1, -1):
                be.fc_bwd_block_reduce(buf, i)
                h = dist.all_reduce_async(buf.bn_sums) if dist.sync_bn else None
                if deferred is not None:
                    dw_and_send(deferred)
                if h is not None:
                    h.wait()
                be.fc_bwd_block_dx(buf, i, gb if dist.sync_bn else buf.B)
                deferred = i
            if deferred is not None:
                dw_and_send(deferred)
            be.fc_bwd_end(buf)
            dist.reduce_gradient_async(self.flat_grads, exclude=self.stacked_grad["w"])
        for p, g in zip(self._param_list, self._grad_views):
            if p.grad is not g:
                p.grad = g

    def forward(self, x, depth=None, objective=None):
        """act_vec [depth+1, B, O].  ``objective`` (probability.HeadObjective, regression with one output) additionally
        runs the likelihood pass inside the head kernels and leaves its results in that object."""
        depth = self.n_layers if depth is None else depth
        if x.dim() == 2 and x.shape[0] == 0 and x.shape[1] == self.input_dim and not self.training:
            return x.new_zeros(depth + 1, 0, self.output_dim, dtype=torch.float32)  # (no rows: nothing to launch)
        if self.training and torch.is_grad_enabled():
            return _FcForward.apply(self, x, depth, objective, *self._param_list)
        return self._run_forward(x, depth, self.training, objective).act

    forward_get_acts = forward


class arq_uncert_fc_MLP(arq_uncert_fc_resnet):
    residual = False
    _block_cls = bern_MLPBlock_nores


class _LnFcForward(torch.autograd.Function):
    """_FcForward for a step whose backward holds no other term of the parameters (the wrappers' captured step).  It hangs on a
    leaf of its own, not on the parameters (whose gradients it writes itself): an act_vec that a caller keeps from before keeps
    the parameters' gradient accumulators alive on its stream, and the backward of a captured step that hung on them would wait for
    them outside the capture, which ends the process.  Next to other terms this node would be wrong: nothing makes autograd run it
    before it adds their gradients, which the trunk's backward then overwrites."""

    @staticmethod
    def forward(ctx, model, x, depth, leaf):
        buf = model._run_forward(x, depth, True)
        ctx.model, ctx.buf, ctx.generation = model, buf, buf.generation
        act, buf.act = buf.act, None  # (a reference cycle through the C++ graph otherwise, as in _FcForward)
        return act

    @staticmethod
    def backward(ctx, dact):
        _FcForward.backward(ctx, dact)
        return None, None, None, None


class arq_uncert_fc_resnet_ln(arq_uncert_fc_resnet):
    """The residual trunk with LayerNorm in its blocks, h + LayerNorm(ReLU(Linear(h))): no counterpart in the reference,
    whose blocks normalise over the batch (src/DUN/layers.py:33-42).

    Rows do not couple: a batch of one row trains, prediction and training compute the same function, and a sharded job
    exchanges gradients and likelihood sums only.  ``act_bits=8`` keeps what the backward reads as 8-bit checkpoints
    (dun_amd.act8), 33 bytes per 32 columns instead of 128: a block's LayerNorm then runs its backward from the checkpoint of the
    rectified Linear output, its Linear's and the head's weight gradients from the checkpoints of the hidden states.
    Same wrappers, flat parameters, optimiser and checkpoints as the BatchNorm trunk.  Weights in float32."""
    _block_cls = bern_LNBlock
    supports_head_objective = False
    _step_alone = False  # set by the wrappers around a captured step

    def __init__(self, input_dim, output_dim, width, n_layers, w_prior=None, BMA_prior=False, act_bits=32):
        if act_bits not in (8, 32):
            raise ValueError("act_bits is 32 or 8 (got %r)" % (act_bits,))
        super(arq_uncert_fc_resnet_ln, self).__init__(input_dim, output_dim, width, n_layers, w_prior, BMA_prior)
        self.act_bits, self.ln_eps = act_bits, 1e-5

    def _flatten(self):
        super(arq_uncert_fc_resnet_ln, self)._flatten()
        if "_nodes" not in self.__dict__:  # autograd nodes of forwards that are alive: the stream of the accumulators they hold
            self._nodes = weakref.WeakKeyDictionary()

    def __getstate__(self):
        st = super(arq_uncert_fc_resnet_ln, self).__getstate__()
        st.pop("_nodes", None)
        return st

    def _flatten_norm(self, dev):
        return None, None, None

    def forward(self, x, depth=None, objective=None):
        if not (self.training and torch.is_grad_enabled() and any(p.requires_grad for p in self._param_list)):
            with torch.no_grad():
                return super(arq_uncert_fc_resnet_ln, self).forward(x, depth, objective)
        if self._step_alone:
            return _LnFcForward.apply(self, x, self.n_layers if depth is None else depth, self.flat_params.new_empty(0).requires_grad_())
        stream = torch.cuda.current_stream(self.flat_params.device) if self.flat_params.is_cuda else None
        # (a live graph keeps the accumulators it found, of a graph before it perhaps, or made on its own stream)
        home = next(iter(list(self._nodes.values())), stream)
        if home != stream and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("an act_vec from before this capture is still alive: its graph holds the parameters' gradient "
                               "accumulators on another stream, and a captured backward would wait for them there; drop it first")
        act = super(arq_uncert_fc_resnet_ln, self).forward(x, depth, objective)
        self._nodes[act.grad_fn] = home
        return act

    forward_get_acts = forward

    def _make_buffers(self, B, depth, train):
        return kernels.backend().ln_fc_buffers(self, B, depth, train)

    def _run_forward(self, x, depth, train, objective=None):
        if x.dim() != 2 or x.shape[1] != self.input_dim:
            raise RuntimeError("expected x of shape [B, %d], got %s" % (self.input_dim, tuple(x.shape)))
        if x.shape[0] == 0:
            raise RuntimeError("an empty batch has nothing to train on")
        be = kernels.backend()
        B, W, O, din = x.shape[0], self.width, self.output_dim, self.input_dim
        x = x.detach().to(torch.float32).contiguous()
        buf = self._get_buffers(B, depth, train)
        buf.generation += 1
        buf.new_act()
        buf.x = x
        p = self.stacked
        be.gemm(x, p["w_in"], B, W, din, bias=p["b_in"], out=buf.h(0))
        if buf.keep8:
            be.act8_pack(buf.h(0), False, out=buf.rows8(buf.Hq, 0))
        if not buf.keep32:
            be.head_forward(buf.h(0), p["w_out"], p["b_out"], out=buf.act[0])
        for i in range(depth):
            h, z = buf.h(i), buf.z(i)
            be.gemm(h, p["w"][i], B, W, W, bias=p["b"][i], out=z)
            # Rectified by the norm that reads it, which keeps NaN: the product's own ReLU makes a NaN 0, and a diverged weight would
            # not show.  The float32 planes that training keeps hold it rectified: a pass in place, 0.2 ms at 65536 x 2048.
            if buf.keep32:
                z.relu_()
            be.layer_norm_forward(z, p["gamma"][i], p["beta"][i], self.ln_eps, res=h, relu=True, want_stats=train,
                                  stats=buf.stats[i] if train else None, out=buf.h(i + 1), pack_x=buf.keep8, pack_y=buf.keep8,
                                  x_packed=buf.rows8(buf.Zq, i), y_packed=buf.rows8(buf.Hq, i + 1))
            if not buf.keep32:
                be.head_forward(buf.h(i + 1), p["w_out"], p["b_out"], out=buf.act[i + 1])
        if buf.keep32:  # every hidden state is there: the shared head over all depths at once
            be.head_forward(buf.H.view((depth + 1) * B, W), p["w_out"], p["b_out"], out=buf.act.view((depth + 1) * B, O))
        return buf

    def _run_backward(self, buf, dact):
        be = kernels.backend()
        buf.ensure_backward(self)
        B, W, O, din, depth = buf.B, self.width, self.output_dim, self.input_dim, buf.depth
        p, g, dist = self.stacked, self.stacked_grad, self._dist
        dact = dact.detach().to(torch.float32).contiguous()
        rows = dact.view((depth + 1) * B, O)
        if buf.keep8:
            be.act8_weight_grad(rows, buf.Hq, W, False, dw=g["w_out"], db=g["b_out"])
        else:
            dw, db, _ = be.head_backward(buf.H.view((depth + 1) * B, W), p["w_out"], rows, need_dH=False)
            g["w_out"].copy_(dw)
            g["b_out"].copy_(db)
        be.gemm(dact[depth], p["w_out"], B, W, O, b_kcontig=False, out=buf.G)
        buf.Wt.copy_(p["w"].transpose(1, 2))
        for k in ("w", "b", "gamma", "beta"):  # blocks past a truncated forward
            if depth < self.n_layers:
                g[k][depth:].zero_()
        sent_from = self.n_layers
        for i in range(depth - 1, -1, -1):
            be.layer_norm_backward(buf.G, None if buf.keep8 else buf.z(i), buf.rows8(buf.Zq, i), p["gamma"][i], buf.stats[i],
                                   relu=True, sums=3, dx=buf.dU, sums_out=buf.sums[i])
            if buf.keep8:
                be.act8_weight_grad(buf.dU, buf.rows8(buf.Hq, i), W, False, want_bias=False, dw=g["w"][i])
            else:
                be.gemm(buf.dU, buf.h(i), W, W, B, a_kcontig=False, b_kcontig=False, splitk_ws=buf.splitk, out=g["w"][i])
            if dist is not None and (sent_from - i >= dist.grad_bucket_blocks or i == 0):
                dist.reduce_gradient_async(g["w"][i:sent_from])
                sent_from = i
            be.gemm(buf.dU, buf.Wt[i], B, W, W, R=buf.G, U=dact[i], V=p["w_out"], out=buf.G)
        if depth:
            g["gamma"][:depth].copy_(buf.sums[:depth, 0])
            g["beta"][:depth].copy_(buf.sums[:depth, 1])
            g["b"][:depth].copy_(buf.sums[:depth, 2])
        be.gemm(buf.G, buf.x, W, din, B, a_kcontig=False, b_kcontig=False, splitk_ws=buf.splitk, out=g["w_in"])
        # (sum_b G: the head's weight gradient of a gradient of ones)
        g["b_in"].copy_(be.head_backward(buf.G, p["w_out"][:1], buf.ones, need_dH=False)[0].view(W))
        if dist is not None:
            if depth == 0 and self.n_layers:
                dist.reduce_gradient_async(g["w"])
            dist.reduce_gradient_async(self.flat_grads, exclude=g["w"])
        for q, gv in zip(self._param_list, self._grad_views):
            if q.grad is not gv:
                q.grad = gv
        self._hold_accumulators()

    def _hold_accumulators(self):
        """A parameter's gradient accumulator runs on the stream that it was made on, by the first of the graphs that have held it since.
        Autograd makes it wait for the gradients that it adds, which may be ready before the trunk's are written, and not for those: it
        waits here."""
        if not self.flat_params.is_cuda or torch.cuda.is_current_stream_capturing():
            return
        current = torch.cuda.current_stream(self.flat_params.device)
        for s in set(self._nodes.values()) - {current}:
            s.wait_stream(current)
