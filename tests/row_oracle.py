"""Layer norm, 8-bit checkpoints and the gradients taken from them, from their formulas in 64 bits on the CPU (tests only)."""
import torch

U32 = 2.0 ** -24  # half a step of float32, relative
HALF = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
GROUP = 32


def codes_of(x, relu):
    """(signed integer codes [rows, G, 32] as float64, exponents [rows, G]; exponent 128 marks a group that is not finite)."""
    v = x.detach().cpu().double()
    if relu:
        v = torch.where(v <= 0, torch.zeros_like(v), v)
    rows, cols = v.shape
    G = (cols + GROUP - 1) // GROUP
    p = torch.zeros(rows, G * GROUP, dtype=torch.float64)
    p[:, :cols] = v
    p = p.view(rows, G, GROUP)
    amax = p.abs().amax(dim=2)  # (NaN stays NaN)
    limit = 255 if relu else 127
    # (amax >= (limit + 1/2) 2^e with e = 121, or 120 rectified, would round to 2^128: no float32)
    bad = ~(amax < (limit + 0.5) * 2.0 ** (120 if relu else 121))
    safe = torch.where(bad | (amax == 0), torch.ones_like(amax), amax)
    e = torch.full_like(safe, -126.0)
    # smallest e >= -126 with rint(amax 2^-e) <= limit, by counting up from below
    guess = torch.floor(torch.log2(safe)) - 10
    e = torch.maximum(e, guess)
    for _ in range(14):
        e = torch.where(torch.round(safe * torch.exp2(-e)) > limit, e + 1, e)
    e = torch.where((amax == 0) & ~bad, torch.full_like(e, -126.0), e)
    q = torch.round(p * torch.exp2(-e).unsqueeze(2))
    if relu:
        q = torch.where(p > 0, q.clamp(min=1), q)
    q = torch.where(bad.unsqueeze(2), torch.zeros_like(q), q)
    e = torch.where(bad, torch.full_like(e, 128.0), e)
    return q, e


def values_of(x, relu):
    q, e = codes_of(x, relu)
    v = q * torch.exp2(e).unsqueeze(2)
    v = torch.where((e == 128).unsqueeze(2), torch.full_like(v, float("nan")), v)
    return v.reshape(x.shape[0], -1)[:, :x.shape[1]]


class Norm(object):
    """Forward and backward in 64 bits, with elementwise bounds on what float32 arithmetic may add.

    A lane adds up to 32 elements of a row one after the other and a tree of at most ten levels adds the lanes (rows
    beyond 32768 elements: cols / 1024 + 16 additions), so a mean is off by at most N u mean|z|, N = 64 or that, and the
    variance and 1 / sqrt by less than 2 N u relative; hence |d xhat| <= N u (r + 2 |xhat|) with r = rstd mean|z|.  The
    remaining operations add a few u each, and the result is rounded once to its type."""

    def __init__(self, x, w, b, eps, res=None, relu=False, bits=None):
        d = lambda t: None if t is None else t.detach().cpu().double()
        self.z = d(x)
        if relu:
            self.z = torch.where(self.z <= 0, torch.zeros_like(self.z), self.z)
        self.relu, self.type = relu, x.dtype
        cols = x.shape[1]
        self.N = max(64, cols // 1024 + 16)
        self.w = torch.ones(cols, dtype=torch.float64) if w is None else d(w)
        b = torch.zeros(cols, dtype=torch.float64) if b is None else d(b)
        res = torch.zeros_like(self.z) if res is None else d(res)
        self.mean = self.z.mean(1, keepdim=True)
        var = ((self.z - self.mean) ** 2).mean(1, keepdim=True)
        self.rstd = 1.0 / torch.sqrt(var + eps)
        xhat = (self.z - self.mean) * self.rstd
        self.r = self.rstd * self.z.abs().mean(1, keepdim=True)
        dxhat = self.N * U32 * (self.r + 2 * xhat.abs())
        self.y = xhat * self.w + b + res
        self.y_tol = dxhat * self.w.abs() + 4 * U32 * ((xhat * self.w).abs() + b.abs() + res.abs()) + self.half(self.y)
        self.seen = values_of(x, relu) if bits == 8 else self.z

    def half(self, t):
        # (a float16 below its smallest normal number rounds to a multiple of 2^-24)
        return HALF[self.type] * t.abs() * (1 + 1e-3) + (2.0 ** -25 if self.type == torch.float16 else 1e-40)

    def backward(self, dy):
        dy = dy.detach().cpu().double()
        xhat = (self.seen - self.mean) * self.rstd
        g = dy * self.w
        m1, m2 = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
        dx = self.rstd * (g - m1 - xhat * m2)
        big = xhat.abs() + self.r + 1e-30
        tol = 4 * self.N * U32 * self.rstd * (g.abs() + g.abs().mean(1, keepdim=True) + big * (g.abs() * big).mean(1, keepdim=True))
        if self.relu:
            dead = self.seen <= 0
            dx = torch.where(dead, torch.zeros_like(dx), dx)
            tol = torch.where(dead, torch.zeros_like(tol), tol)
        self.dx, self.dx_tol = dx, tol + self.half(dx)
        # column sums: at most 128 additions one after the other (a team's rows, the waves, the partial rows)
        rows = dy.shape[0]
        n = 128 + rows // 512
        self.dw, self.db, self.ds = (dy * xhat).sum(0), dy.sum(0), dx.sum(0)
        self.dw_tol = (n + 3 * self.N) * U32 * (dy.abs() * big).sum(0) + 1e-30
        self.db_tol = n * U32 * dy.abs().sum(0) + 1e-30
        self.ds_tol = tol.sum(0) + n * U32 * dx.abs().sum(0) + 1e-30
        return self


def within(got, want, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), "%s: %d of %d off, worst %.3g times its bound" % (
        what, int(bad.sum()), bad.numel(), float(((got - want).abs() / tol)[bad].max()))
