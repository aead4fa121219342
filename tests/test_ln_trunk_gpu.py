"""The LayerNorm trunk on the GPU: forward and gradients against 64-bit formulas, the wrappers around it, and the row operators
used together as a block uses them."""
import contextlib
import io
import subprocess
import sys

import numpy as np
import pytest
import torch

from oracle import dun_oracle as O
from tests.row_oracle import Norm, values_of

pytestmark = pytest.mark.gpu


def build(din=13, outs=1, W=100, L=4, bits=32, vi=True, regression=True, N=455, seed=0, lr=1e-2):
    from dun_amd.probability import depth_categorical, depth_categorical_VI
    from dun_amd.stochastic_fc_models import arq_uncert_fc_resnet_ln
    from dun_amd.training_wrappers import DUN, DUN_VI
    torch.manual_seed(seed)
    prior = [1.0 / (L + 1)] * (L + 1)
    with contextlib.redirect_stdout(io.StringIO()):
        model = arq_uncert_fc_resnet_ln(din, outs, W, L, act_bits=bits)
        pm = (depth_categorical_VI if vi else depth_categorical)(prior, cuda=True)
        return (DUN_VI if vi else DUN)(model, pm, N, lr=lr, momentum=0.5, cuda=True, regression=regression)


def near(got, want, rel, what):
    got, want = got.detach().cpu().double(), want.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    err = float((got - want).norm() / (want.norm() + 1e-30))
    assert err <= rel, "%s: %.3g off, %.3g allowed" % (what, err, rel)


def decoded(packed, cols, relu):
    """Values of codes and exponents, from their definition."""
    codes, exps = (t.cpu().double() for t in packed)
    return ((codes - (0 if relu else 128)) * torch.exp2(exps - 127).repeat_interleave(32, dim=1))[:, :cols]


def formulas(model, x, dact, H, Z, seen_h, seen_z):
    """Backward in 64 bits from given hidden states H[d] and rectified Linear outputs Z[i], where the gradients are taken from
    seen_h and seen_z (the same, or the values of their checkpoints): {parameter kind: gradient}."""
    d = lambda t: t.detach().cpu().double()
    p = {k: d(v) for k, v in model.stacked.items()}
    dact = d(dact)
    L = model.n_layers
    g = {k: torch.zeros_like(v) for k, v in p.items()}
    g["w_out"] = sum(dact[i].t() @ seen_h[i] for i in range(L + 1))
    g["b_out"] = dact.sum((0, 1))
    G = dact[L] @ p["w_out"]
    for i in range(L - 1, -1, -1):
        n = Norm(Z[i], p["gamma"][i], p["beta"][i], model.ln_eps, None, True)
        n.seen = seen_z[i]
        n.backward(G)
        g["gamma"][i], g["beta"][i], g["b"][i] = n.dw, n.db, n.ds
        g["w"][i] = n.dx.t() @ seen_h[i]
        G = G + n.dx @ p["w"][i] + dact[i] @ p["w_out"]
    g["w_in"], g["b_in"] = G.t() @ d(x), G.sum(0)
    return g


# A product of K terms in float32 is off by about sqrt(K) u relative to its norm, K <= 2048 rows or columns here: 3e-6; a gradient passes
# up to 3 products and a norm per block and up to 6 blocks, each amplifying what came before by a little over 1: 1e-4 holds them all
REL = 1e-4


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("B,din,outs,W,L", [(1, 3, 1, 8, 2), (7, 1, 1, 33, 3), (128, 13, 1, 100, 6), (300, 64, 10, 257, 3), (513, 4, 2, 512, 2),
                                            (2048, 64, 1, 1024, 2), (64, 5, 1, 16, 0)])
def test_forward_and_gradients(B, din, outs, W, L, bits):
    model = build(din, outs, W, L, bits).model.train()
    with torch.no_grad():
        for k in ("gamma", "beta", "b"):
            model.stacked[k].add_(0.1 * torch.randn_like(model.stacked[k]))
    x = torch.randn(B, din, device="cuda")
    dact = torch.randn(L + 1, B, outs, device="cuda") / B
    act = model(x)
    buf = next(iter(model._fc_cache.values()))
    # the function itself, in 64 bits
    p = {k: v.detach().cpu().double() for k, v in model.stacked.items()}
    h = x.cpu().double() @ p["w_in"].t() + p["b_in"]
    want = [h @ p["w_out"].t() + p["b_out"]]
    for i in range(L):
        z = torch.relu(h @ p["w"][i].t() + p["b"][i])
        h = Norm(z, p["gamma"][i], p["beta"][i], model.ln_eps, h).y
        want.append(h @ p["w_out"].t() + p["b_out"])
    near(act, torch.stack(want), REL, "act")
    act.backward(dact)
    # the states from a float32 trunk of the same parameters.  (Its planes of an odd width are aligned differently, which takes other product
    # kernels and may change last bits, and with them, rarely, a code: the checkpoints' values are the trunk's own)
    twin = build(din, outs, W, L, 32).model.train()
    twin.flat_params.copy_(model.flat_params)
    act2 = twin(x)
    near(act, act2, 1e-6, "act of the two trunks")
    tb = next(iter(twin._fc_cache.values()))
    H, Z = [tb.H[i].cpu().double() for i in range(L + 1)], [tb.Z[i].cpu().double() for i in range(L)]
    seen_h, seen_z = H, Z
    if bits == 8:
        seen_h = [decoded(buf.rows8(buf.Hq, i), W, False) for i in range(L + 1)]
        seen_z = [decoded(buf.rows8(buf.Zq, i), W, True) for i in range(L)]
        for got, t, relu in [(v, tb.H[i], False) for i, v in enumerate(seen_h)] + [(v, tb.Z[i], True) for i, v in enumerate(seen_z)]:
            near(got, values_of(t, relu), 1e-3, "values of a checkpoint")
    g = formulas(model, x, dact, H, Z, seen_h, seen_z)
    for k, v in model.stacked_grad.items():
        if v.numel():
            near(v, g[k], REL, k)
    if bits == 8:
        assert buf.H.shape[0] == 1 and buf.Hq[0].shape[0] == (L + 1) * B


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("vi,regression", [(True, True), (False, True), (True, False)])
def test_fit_graphed_and_eager_agree(bits, vi, regression, monkeypatch):
    outs = 1 if regression else 4
    x, y = O.synthetic_regression(200, 13, seed=1)
    if not regression:
        y = (torch.as_tensor(x)[:, 0] > 0).long() + 2 * (torch.as_tensor(x)[:, 1] > 0).long()
    runs = []
    for eager in (False, True):
        if eager:
            monkeypatch.setenv("DUN_NO_GRAPH", "1")
        net = build(outs=outs, bits=bits, vi=vi, regression=regression)
        out = [net.fit(x, y) for _ in range(6)]
        if not eager:
            assert any(s["graph"] is not None for s in net._graph_states.values())
        runs.append((out, net.model.flat_params.clone(), net.eval(x, y)))
    assert np.array_equal(np.array(runs[0][0]), np.array(runs[1][0])) and torch.equal(runs[0][1], runs[1][1])
    assert np.isfinite(np.array(runs[0][0])).all() and runs[0][2] == runs[1][2]


def test_two_batch_sizes_alternate_in_graphs():
    x, y = O.synthetic_regression(300, 13, seed=2)
    runs = []
    for eager in (False, True):
        net = build(bits=8)
        net.graph_steps = not eager
        out = []
        for _ in range(4):
            out += [net.fit(x[:200], y[:200]), net.fit(x[200:], y[200:])]
        runs.append((out, net.model.flat_params.clone()))
    assert runs[0][0] == runs[1][0] and torch.equal(runs[0][1], runs[1][1])


def test_prediction_keeps_nothing_and_needs_no_batch():
    net = build(W=256, L=3, bits=8)
    x, y = O.synthetic_regression(400, 13, seed=3)
    net.fit(x, y)
    mu, std = net.predict(x, get_std=True)
    assert mu.shape == (400, 1) and torch.isfinite(std).all()
    one = torch.cat([net.predict(x[i:i + 1]) for i in range(5)])
    near(one, mu[:5], 1e-5, "rows by themselves")  # (other product kernels for one row: sums in another order)
    b = net.model._get_buffers(400, 3, False)
    assert b.H.shape[0] == 1 and b.Z.shape[0] == 1 and b.Hq is None and b.stats is None
    assert net.predict(torch.as_tensor(x)[:0]).shape == (0, 1)


def test_checkpoint_roundtrip(tmp_path):
    x, y = O.synthetic_regression(150, 13, seed=4)
    net = build(bits=8)
    net.fit(x, y)
    with contextlib.redirect_stdout(io.StringIO()):
        net.save_state(str(tmp_path / "s.pt"))
        net.save(str(tmp_path / "s.dat"))
        a, b = build(bits=8, seed=5), build(bits=8, seed=6)
        a.load_state(str(tmp_path / "s.pt"))
        b.load(str(tmp_path / "s.dat"))
    want = [net.fit(x, y) for _ in range(3)]
    assert [a.fit(x, y) for _ in range(3)] == want and [b.fit(x, y) for _ in range(3)] == want


def test_eight_bits_hold_a_quarter_of_the_activations():
    sizes = {}
    for bits in (32, 8):
        model = build(64, 1, 512, 8, bits).model.train()
        model(torch.randn(2048, 64, device="cuda"))
        b = next(iter(model._fc_cache.values()))
        sizes[bits] = sum(t.numel() * t.element_size() for t in (b.H, b.Z) + ((b.Hq + b.Zq) if b.Hq is not None else ()))
    assert sizes[8] <= 0.4 * sizes[32]  # (two float32 planes of 17 stay; the rest at 33 / 128)


def test_a_block_from_the_public_operators_matches_the_trunk():
    """Linear -> ReLU -> LayerNorm -> residual from act8.linear and layer_norm, autograd around them: the gradients of the
    trunk with 8-bit checkpoints."""
    from dun_amd import act8
    from dun_amd.layer_norm import layer_norm
    model = build(6, 1, 96, 2, bits=8).model.train()
    x = torch.randn(77, 6, device="cuda")
    dact = torch.randn(3, 77, 1, device="cuda")
    act = model(x)
    act.backward(dact)
    leaves = {n: p.detach().clone().requires_grad_() for n, p in model.named_parameters()}
    h = torch.nn.functional.linear(x, leaves["input_layer.weight"], leaves["input_layer.bias"])
    packed, out = act8.pack(h), []
    head = lambda t, q: act8.linear(t, leaves["output_layer.weight"], leaves["output_layer.bias"], q)
    out.append(head(h, packed))
    for i in range(2):
        n = "stochstic_layers.%d.block." % i
        u = act8.linear(h, leaves[n + "0.weight"], leaves[n + "0.bias"], packed)
        h, packed = layer_norm(u, leaves[n + "2.weight"], leaves[n + "2.bias"], 1e-5, residual=h, relu=True, bits=8, pack_output=True)
        out.append(head(h, packed))
    near(torch.stack(out), act, 1e-6, "act")
    grads = torch.autograd.grad(torch.stack(out), list(leaves.values()), dact)
    for (n, p), g in zip(model.named_parameters(), grads):
        # (a hidden state that differs in its last bit may take the neighbouring code: one of 77 * 96 elements by 1 %)
        near(p.grad, g, 1e-3, n)


@pytest.mark.parametrize("bits", ["32", "8"])
def test_the_toy_command_trains_it(bits, tmp_path):
    r = subprocess.run([sys.executable, "examples/train_toy.py", "--n_epochs", "6", "--network", "ResNetLN", "--act_bits", bits, "--N_layers", "3",
                        "--width", "32", "--savedir", str(tmp_path)], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "final ELBO estimate" in r.stdout, r.stderr[-2000:]


def test_a_kept_act_vec_does_not_disturb_a_captured_step():
    x, y = O.synthetic_regression(200, 13, seed=7)
    runs = []
    for keep in (False, True):
        net = build(bits=8)
        net.model.train()
        kept = net.model(torch.as_tensor(x).cuda()) if keep else None
        runs.append([net.fit(x, y) for _ in range(4)])
        assert any(s["graph"] is not None for s in net._graph_states.values())
        if keep:
            with pytest.raises(RuntimeError, match="reused by a later"):
                kept.sum().backward()
    assert runs[0] == runs[1]


def test_frozen_parameters_need_no_gradient():
    m = build().model.train()
    x = torch.randn(8, 13, device="cuda")
    assert m(x).requires_grad
    for p in m.parameters():
        p.requires_grad_(False)
    assert not m(x).requires_grad
