"""Layer normalisation, 8-bit activation checkpoints and the gradients that are taken from them: cases, plain forms and
the calls that a program makes of them.

What the operators compute (x, u, h, dy: [rows, cols], row-major):

  norm    y = (x - mean) * rstd * w + b per row, rstd = 1 / sqrt(var + eps) with the biased variance; in training also
          g = dy * w, xhat = (x - mean) * rstd, dx = rstd * (g - mean(g) - xhat * mean(g * xhat)), dw = sum_rows dy * xhat,
          db = sum_rows dy.
  norm8   the residual block's form, y = h + norm(max(u, 0)), whose backward reads max(u, 0) from its 8-bit checkpoint:
          xhat = (value - mean) * rstd with the forward's mean and rstd, du = dx where value > 0 and 0 elsewhere.
  pack    an 8-bit checkpoint and the values that it stands for.  Groups of 32 consecutive columns of a row share a
          scale 2^e, e the smallest integer (not below -126) for which the group's largest magnitude rounds to at most
          127 (255 for a rectified input, whose codes are unsigned): value = 2^e * rint(x * 2^-e).  A positive element of a
          rectified input keeps a code of at least 1, so that value > 0 exactly where the input was.
  grad8   a Linear layer's weight and bias gradient with its input taken from a checkpoint: dw = dy^T value, db = sum_rows dy.
"""
import math

import torch

own = False

EPS = 1e-5
GROUP = 32
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # one row of a toy / UCI regression net (10 blocks of width 100) at prediction time: latency alone
        {"name": "norm predict 1x100", "op": "norm", "rows": 1, "cols": 100, "type": "fp32", "train": False},
        # one block of that net in training, batch 512
        {"name": "norm train 512x100", "op": "norm", "rows": 512, "cols": 100, "type": "fp32", "train": True},
        # the wide MLP (width 2048, batch 65536): streaming, far larger than the caches
        {"name": "norm train 65536x2048", "op": "norm", "rows": 65536, "cols": 2048, "type": "fp32", "train": True},
        # 16-bit features of a ragged batch with an odd width: no row but the first is aligned
        {"name": "norm train bf16 16391x1031", "op": "norm", "rows": 16391, "cols": 1031, "type": "bf16", "train": True},
        # the residual block of the small net
        {"name": "norm8 512x100", "op": "norm8", "rows": 512, "cols": 100, "type": "fp32"},
        # an odd width and batch between the two nets
        {"name": "norm8 4099x517", "op": "norm8", "rows": 4099, "cols": 517, "type": "fp32"},
        # the residual block of the wide MLP, where the checkpoints save most
        {"name": "norm8 65536x2048", "op": "norm8", "rows": 65536, "cols": 2048, "type": "fp32"},
        # a ragged 16-bit activation: groups that end inside a row, rows that start anywhere
        {"name": "pack fp16 1537x1001", "op": "pack", "rows": 1537, "cols": 1001, "type": "fp16", "relu": True},
        # the wide MLP's hidden state, signed
        {"name": "pack 65536x2048", "op": "pack", "rows": 65536, "cols": 2048, "type": "fp32", "relu": False},
        # a Linear layer of the small net
        {"name": "grad8 512x100x100", "op": "grad8", "rows": 512, "outs": 100, "cols": 100, "type": "fp32", "relu": False},
        # the shared output layer over 12 exits of a batch of 4096: ten classes, 2048 pooled features
        {"name": "grad8 49152x10x2048", "op": "grad8", "rows": 49152, "outs": 10, "cols": 2048, "type": "fp32", "relu": True},
        # a Linear layer of the wide MLP: the largest product
        {"name": "grad8 65536x2048x2048", "op": "grad8", "rows": 65536, "outs": 2048, "cols": 2048, "type": "fp32", "relu": False},
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 0.5 / hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm8", "pack", "grad8", "grad8"])
    kind = rng.choice(["fp32", "fp32", "bf16", "fp16"])
    most = 65536 * 2048
    cols = _spread(rng, 1, 8192 if op != "grad8" else 2048)
    rows = _spread(rng, 1, min(65536, most // cols))
    case = {"op": op, "rows": rows, "cols": cols, "type": kind}
    if op == "norm":
        case["train"] = rng.random() < 0.7
    elif op == "pack":
        case["relu"] = rng.random() < 0.5
    elif op == "grad8":
        case["outs"] = _spread(rng, 1, 2048)
        case["relu"] = rng.random() < 0.5
    return case


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rows, cols, kind = case["rows"], case["cols"], TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)

    state = {"case": case}
    if case["op"] in ("norm", "norm8"):
        # a hidden state: every row has its own mean and spread, every column its own offset
        x = normal(rows, cols) * (0.5 + normal(rows, 1).abs()) + 0.5 * normal(rows, 1) + 0.3 * normal(cols)
        state["x"] = x.to(kind)
        state["w"] = 1.0 + 0.2 * normal(cols)
        state["b"] = 0.1 * normal(cols)
        if case["op"] == "norm8" or case["train"]:
            state["dy"] = normal(rows, cols).to(kind)
        if case["op"] == "norm8":
            state["h"] = normal(rows, cols).to(kind)
        return state
    x = normal(rows, cols) * (0.5 + normal(rows, 1).abs()) + 0.3 * normal(cols)
    x = x.to(kind if case["op"] == "pack" else torch.float32)
    if case["op"] == "pack":
        state["x"] = x
        return state
    # the gradient of a mean over the batch: small, of very different sizes from row to row
    state["dy"] = (normal(rows, case["outs"]) * torch.exp(normal(rows, 1)) / max(1.0, rows ** 0.5)).to(kind)
    if own:
        from dun_amd import act8
        state["packed"] = act8.pack(x, relu=case["relu"])
    else:
        state["packed"] = _pack(x, case["relu"])
    return state


# ---- plain forms -------------------------------------------------------------------------------------------------------
def _scale(byte):
    """2^(byte - 127) from a biased exponent: the bits of a float."""
    return (byte.to(torch.int32) << 23).view(torch.float32)


def _pack(x, relu):
    """(codes [rows, groups, 32] as floats, biased exponents [rows, groups, 1])"""
    rows, cols = x.shape
    groups = (cols + GROUP - 1) // GROUP
    v = torch.zeros(rows, groups * GROUP, device=x.device, dtype=torch.float32)
    v[:, :cols] = x.float().clamp(min=0) if relu else x.float()
    v = v.view(rows, groups, GROUP)
    mant, power = torch.frexp(v.abs().amax(dim=2, keepdim=True))  # amax = mant * 2^power, mant in [0.5, 1)
    top = 8 if relu else 7
    edge = (255.5 / 256.0) if relu else (127.5 / 128.0)
    byte = (power - top + (mant >= edge).to(power.dtype) + 127).clamp(min=1)
    codes = torch.round(v * _scale(254 - byte))
    if relu:
        codes = torch.where(v > 0, codes.clamp(min=1), codes)
    return codes.to(torch.uint8 if relu else torch.int8), byte.to(torch.uint8)


def _unpack(packed, cols):
    codes, byte = packed
    v = codes.float() * _scale(byte)
    return v.view(codes.shape[0], -1)[:, :cols]


def _norm(x, w, b):
    mean = x.mean(dim=1, keepdim=True)
    c = x - mean
    rstd = 1.0 / torch.sqrt((c * c).mean(dim=1, keepdim=True) + EPS)
    return c * rstd * w + b, mean, rstd


def _norm_grad(dy, x, w, mean, rstd):
    xhat = (x - mean) * rstd
    g = dy * w
    dx = rstd * (g - g.mean(dim=1, keepdim=True) - xhat * (g * xhat).mean(dim=1, keepdim=True))
    return dx, (dy * xhat).sum(dim=0), dy.sum(dim=0)


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_plain(state):
    case = state["case"]
    kind = TYPES[case["type"]]
    if case["op"] == "norm":
        x = state["x"].float()
        y, mean, rstd = _norm(x, state["w"], state["b"])
        if not case["train"]:
            return y.to(kind)
        dx, dw, db = _norm_grad(state["dy"].float(), x, state["w"], mean, rstd)
        return y.to(kind), dx.to(kind), dw, db
    if case["op"] == "norm8":
        z = state["x"].float().clamp(min=0)
        y, mean, rstd = _norm(z, state["w"], state["b"])
        value = _unpack(_pack(z, True), case["cols"])
        dx, dw, db = _norm_grad(state["dy"].float(), value, state["w"], mean, rstd)
        return (y + state["h"].float()).to(kind), torch.where(value > 0, dx, torch.zeros_like(dx)).to(kind), dw, db
    if case["op"] == "pack":
        return _unpack(_pack(state["x"], case["relu"]), case["cols"]).contiguous()
    dy = state["dy"].float()
    return dy.t() @ _unpack(state["packed"], case["cols"]), dy.sum(dim=0)


# ---- the framework's operators -------------------------------------------------------------------------------------------
def _run_own(state):
    from dun_amd import act8
    from dun_amd.layer_norm import layer_norm, layer_norm_backward, layer_norm_forward
    case = state["case"]
    if case["op"] == "norm":
        if not case["train"]:
            return layer_norm(state["x"], state["w"], state["b"], EPS)
        y, saved = layer_norm_forward(state["x"], state["w"], state["b"], EPS)
        dx, dw, db = layer_norm_backward(state["dy"], saved)
        return y, dx, dw, db
    if case["op"] == "norm8":
        y, saved = layer_norm_forward(state["x"], state["w"], state["b"], EPS, residual=state["h"], relu=True, bits=8)
        dx, dw, db = layer_norm_backward(state["dy"], saved)
        return y, dx, dw, db
    if case["op"] == "pack":
        return act8.pack(state["x"], relu=case["relu"]).unpack()
    return act8.weight_grad(state["dy"], state["packed"])


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def _exact_values(x, relu):
    v = x.double()
    if relu:
        v = torch.relu(v)
    rows, cols = v.shape
    out = torch.empty_like(v)
    limit = 255 if relu else 127
    for at in range(0, cols, GROUP):
        part = v[:, at:at + GROUP]
        big = part.abs().max(dim=1, keepdim=True).values
        e = torch.floor(torch.log2(torch.where(big > 0, big, torch.ones_like(big)))) - (9 if relu else 8)
        for _ in range(4):
            e = torch.where(torch.round(big * torch.exp2(-e)) > limit, e + 1, e)
        step = torch.exp2(e.clamp(min=-126))
        q = torch.round(part / step)
        if relu:
            q = torch.maximum(q, (part > 0).double())
        out[:, at:at + GROUP] = q * step
    return out


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "pack":
        return _exact_values(s["x"], case["relu"])
    if case["op"] == "grad8":
        codes, byte = s["packed"]
        value = torch.ldexp(codes.double(), byte.double() - 127).reshape(case["rows"], -1)[:, :case["cols"]]
        dy = s["dy"].double()
        return dy.t() @ value, dy.sum(0)
    x = s["x"].double()
    if case["op"] == "norm8":
        x = torch.relu(x)
    w, b = s["w"].double(), s["b"].double()
    var, mean = torch.var_mean(x, dim=1, keepdim=True, unbiased=False)
    rstd = torch.rsqrt(var + EPS)
    y = (x - mean) * rstd * w + b
    if case["op"] == "norm8":
        y = y + s["h"].double()
    elif not case["train"]:
        return y
    seen = _exact_values(s["x"], True) if case["op"] == "norm8" else x
    xhat = (seen - mean) * rstd
    dy = s["dy"].double()
    g = dy * w
    n = case["cols"]
    dx = (g * n - g.sum(1, keepdim=True) - xhat * (g * xhat).sum(1, keepdim=True)) * (rstd / n)
    if case["op"] == "norm8":
        dx = dx * (seen > 0)
    return y, dx, (dy * xhat).sum(0), dy.sum(0)


def work(case):
    n, size = case["rows"] * case["cols"], SIZE[case["type"]]
    if case["op"] == "norm":
        if not case["train"]:
            return {"bytes": 2 * n * size + 8 * case["cols"], "flops": 8 * n}
        return {"bytes": 4 * n * size + 16 * case["cols"], "flops": 20 * n}
    if case["op"] == "norm8":
        return {"bytes": 5 * n * size + 16 * case["cols"], "flops": 26 * n}
    if case["op"] == "pack":
        return {"bytes": n * (size + 4), "flops": 4 * n}
    groups = (case["cols"] + GROUP - 1) // GROUP
    product = case["rows"] * case["outs"]
    return {"bytes": n + case["rows"] * groups + product * size + 4 * case["outs"] * (case["cols"] + 1),
            "flops": 2 * product * case["cols"] + product}
