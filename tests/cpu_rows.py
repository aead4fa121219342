"""TEST INFRASTRUCTURE: the CPU stand-in of tests/cpu_backend.py with the row operators (products, layer norm, 8-bit
checkpoints) that the LayerNorm trunk asks its backend for, in plain torch."""
import torch
import torch.nn.functional as F

from dun_amd.kernels import LnFcBuffers
from tests.cpu_backend import CpuBackend
from tests.row_oracle import codes_of


class CpuRowBackend(CpuBackend):
    def act8_buffers(self, rows, cols, device):
        groups = (cols + 31) // 32
        return torch.zeros(rows, groups * 32, dtype=torch.uint8), torch.zeros(rows, groups, dtype=torch.uint8)

    def act8_pack(self, x, relu, out=None):
        q, e = codes_of(x, relu)
        codes, exps = self.act8_buffers(x.shape[0], x.shape[1], None) if out is None else out
        codes.copy_((q + (0 if relu else 128)).reshape(codes.shape))
        exps.copy_(e + 127)
        return codes, exps

    def _values(self, packed, cols, relu):
        codes, exps = packed
        v = (codes.double() - (0 if relu else 128)) * torch.exp2(exps.double() - 127).repeat_interleave(32, dim=1)
        return v[:, :cols].float()

    def act8_weight_grad(self, dy, packed, cols, relu, want_bias=True, dw=None, db=None):
        got = dy.t() @ self._values(packed, cols, relu)
        dw = got if dw is None else dw.copy_(got)
        if want_bias or db is not None:
            db = dy.sum(0) if db is None else db.copy_(dy.sum(0))
        return dw, db

    def layer_norm_forward(self, x, w, b, eps, res=None, relu=False, want_stats=True, pack_x=False, pack_y=False, out=None,
                           stats=None, x_packed=None, y_packed=None):
        z = torch.relu(x) if relu else x
        mean = z.mean(1)
        rstd = 1 / torch.sqrt(z.var(1, unbiased=False) + eps)
        y = (z - mean[:, None]) * rstd[:, None] * w + b
        y = y if res is None else y + res
        if stats is not None:
            stats[0], stats[1] = mean, rstd
        if pack_x:
            self.act8_pack(z, relu, out=x_packed)
        y = y if out is None else out.copy_(y)
        if pack_y:
            self.act8_pack(y, False, out=y_packed)
        return y, stats, x_packed, y_packed

    def layer_norm_backward(self, dy, x, packed, w, stats, relu=False, sums=2, dx=None, sums_out=None):
        z = self._values(packed, dy.shape[1], relu) if x is None else (torch.relu(x) if relu else x)
        xhat = (z - stats[0][:, None]) * stats[1][:, None]
        g = dy * w
        d = stats[1][:, None] * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        d = torch.where(z <= 0, torch.zeros_like(d), d) if relu else d
        sums_out[0], sums_out[1], sums_out[2] = (dy * xhat).sum(0), dy.sum(0), d.sum(0)
        return dx.copy_(d), sums_out

    def gemm(self, A, B, M, N, K, a_kcontig=True, b_kcontig=True, bias=None, relu=False, R=None, U=None, V=None,
             colstats=False, out=None, splitk_ws=None, bn=None):
        C = (A if a_kcontig else A.t()) @ (B.t() if b_kcontig else B)
        assert C.shape == (M, N) and (A.shape[1] if a_kcontig else A.shape[0]) == K
        C = C if bias is None else C + bias
        C = torch.relu(C) if relu else C
        C = C if U is None else C + U @ V
        C = C if R is None else C + R
        return C if out is None else out.copy_(C)

    def head_forward(self, H, w, b, out=None):
        y = F.linear(H, w, b)
        return y if out is None else out.copy_(y)

    def ln_fc_buffers(self, model, B, depth, train):
        return LnFcBuffers(model, B, depth, train)
