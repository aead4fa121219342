"""Gradients of the LayerNorm trunk beside other terms of the same parameters: a weight prior, a penalty, an ELBO that is differentiated as
a whole.  The trunk writes its parameters' gradients itself and autograd adds the other terms' to them, so the sum has to be the
float32 sum of the two, to the bit, in whichever order the terms were recorded."""
import contextlib
import io

import pytest
import torch

DEVICES = [pytest.param("cpu", id="cpu"), pytest.param("cuda", marks=pytest.mark.gpu, id="gpu")]


@pytest.fixture(params=DEVICES)
def dev(request):
    from dun_amd import kernels
    if request.param == "cpu":
        from tests.cpu_rows import CpuRowBackend
        kernels.set_backend(CpuRowBackend())
        yield "cpu"
        kernels.set_backend(None)
    else:
        yield "cuda"


def build(dev, bits, w_prior=None, regression=True, W=40, L=3):
    from dun_amd.probability import depth_categorical_VI
    from dun_amd.stochastic_fc_models import arq_uncert_fc_resnet_ln
    from dun_amd.training_wrappers import DUN_VI
    torch.manual_seed(0)
    with contextlib.redirect_stdout(io.StringIO()):
        model = arq_uncert_fc_resnet_ln(5, 1 if regression else 4, W, L, w_prior=w_prior, act_bits=bits)
        pm = depth_categorical_VI([1.0 / (L + 1)] * (L + 1), cuda=dev == "cuda")
        return DUN_VI(model, pm, 300, lr=1e-2, momentum=0.5, cuda=dev == "cuda", regression=regression)


def penalty(model):
    return sum((p ** 2).sum() + p.sum() for p in model.parameters())


def alone(model, x, dact, term):
    """{parameter name: the trunk's gradient + the term's}, each taken by itself."""
    model(x).backward(dact)
    mine = {n: p.grad.clone() for n, p in model.named_parameters()}
    other = torch.autograd.grad(term(), list(model.parameters()), allow_unused=True)
    return {n: g if o is None else g + o for (n, g), o in zip(mine.items(), other)}


def same(model, want):
    for n, p in model.named_parameters():
        assert torch.equal(p.grad, want[n]), n
    for p, g in zip(model._param_list, model._grad_views):
        assert p.grad is g


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("order", ["trunk first", "penalty first"])
def test_a_penalty_on_the_parameters(dev, bits, order):
    m = build(dev, bits).model.train()
    x, dact = torch.randn(33, 5, device=dev), torch.randn(4, 33, 1, device=dev)
    want = alone(m, x, dact, lambda: penalty(m))
    for _ in range(2):
        if order == "trunk first":
            act = m(x)
            pen = penalty(m)
        else:
            pen = penalty(m)
            act = m(x)
        torch.autograd.backward([act, pen], [dact, torch.ones_like(pen)])
        same(m, want)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("regression", [True, False])
@pytest.mark.parametrize("order", ["trunk first", "prior first"])
def test_an_elbo_with_a_weight_prior(dev, bits, regression, order):
    from dun_amd.probability import diag_w_Gauss_loglike
    net = build(dev, bits, diag_w_Gauss_loglike(0, 0.3), regression)
    m, pm, lik = net.model.train(), net.prob_model, net.f_neg_loglike
    x = torch.randn(48, 5, device=dev)
    y = torch.randn(48, 1, device=dev) if regression else torch.randint(0, 4, (48,), device=dev)
    elbo = lambda prior, act: -pm.estimate_ELBO(prior, act, y, lik, 300) / 300
    leaf = m(x).detach().requires_grad_()
    dact = torch.autograd.grad(elbo(m.get_w_prior_loglike().detach(), leaf), leaf)[0]
    want = alone(m, x, dact, lambda: elbo(m.get_w_prior_loglike(), leaf.detach()))
    without = {n: p.grad.clone() for n, p in m.named_parameters()}
    if order == "trunk first":
        act = m(x)
        prior = m.get_w_prior_loglike()
    else:
        prior = m.get_w_prior_loglike()
        act = m(x)
    elbo(prior, act).backward()
    same(m, want)
    w = m.input_layer.weight
    assert not torch.equal(w.grad, without["input_layer.weight"])


@pytest.mark.parametrize("bits", [32, 8])
def test_fit_with_a_weight_prior(dev, bits):
    """The wrapper takes the prior's backward by itself, behind the trunk's: the same step as an ELBO differentiated as a whole."""
    from dun_amd.probability import diag_w_Gauss_loglike
    x, y = torch.randn(48, 5), torch.randn(48, 1)
    a, b = build(dev, bits, diag_w_Gauss_loglike(0, 0.3)), build(dev, bits, diag_w_Gauss_loglike(0, 0.3))
    a.fit(x, y)
    b.model.train()
    prior = b.model.get_w_prior_loglike()
    elbo = b.prob_model.estimate_ELBO(prior, b.model(x.to(dev)), y.to(dev), b.f_neg_loglike, 300)
    (-elbo / 300).backward()
    g = b.model.flat_grads.clone()
    b.optimizer.step()
    p, q = a.model.flat_params, b.model.flat_params
    # one step of lr 1e-2: the gradients' difference (scaled by the depth weights and 1 / N in another order, then at most 12
    # products of up to 48 terms and 3 norms: 1e-4 relative) and one rounding of the parameters
    assert (p - q).norm() <= 1e-2 * 1e-4 * g.norm() + 2.0 ** -23 * p.norm()


def test_every_parameter_is_told_of_its_gradient(dev):
    m = build(dev, 8).model.train()
    told = []
    for n, p in m.named_parameters():
        p.register_post_accumulate_grad_hook(lambda q, n=n: told.append(n))
    (m(torch.randn(9, 5, device=dev)).sum() + penalty(m)).backward()
    assert sorted(told) == sorted(n for n, _ in m.named_parameters())


def test_nodes_are_forgotten_with_their_graphs(dev):
    m = build(dev, 8).model.train()
    act = m(torch.randn(9, 5, device=dev))
    assert len(m._nodes) == 1
    loss = act.sum()
    del act
    assert len(m._nodes) == 1
    loss.backward()
    del loss
    assert len(m._nodes) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_of_ones_own_with_a_penalty(bits):
    m = build("cuda", bits).model.train()
    x, dact = torch.randn(33, 5, device="cuda"), torch.randn(4, 33, 1, device="cuda")

    def step():
        pen = penalty(m)
        act = m(x)
        torch.autograd.backward([act, pen], [dact, torch.ones_like(pen)])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    assert len(m._nodes) == 0  # (no graph of the same parameters is alive)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(4):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
            m.flat_grads.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        got = m.flat_grads.clone()
        want = alone(m, x, dact, lambda: penalty(m))
        for n, p in m.named_parameters():
            at = next(g for q, g in zip(m._param_list, m._grad_views) if q is p)
            k = at.storage_offset()
            assert torch.equal(got[k:k + at.numel()].view(at.shape), want[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("dropped", [False, True])
@pytest.mark.parametrize("kept_on", ["side", "default"])
def test_an_older_graph_on_another_stream(kept_on, dropped):
    """The parameters' accumulators belong to the older graph's stream; the penalty's gradients are ready before the trunk's are written (the hook
    holds the trunk's backward back on its stream)."""
    m = build("cuda", 8).model.train()
    x, dact = torch.randn(33, 5, device="cuda"), torch.randn(4, 33, 1, device="cuda")
    want = alone(m, x, dact, lambda: penalty(m))
    default, side = torch.cuda.current_stream(), torch.cuda.Stream()
    old, new = (side, default) if kept_on == "side" else (default, side)
    side.wait_stream(default)
    with torch.cuda.stream(old):
        kept = m(x)
    new.wait_stream(old)
    with torch.cuda.stream(new):
        act = m(x)
        if dropped:  # (the accumulators live on in the graph that found them)
            kept = None
        act.register_hook(lambda g: (torch.cuda._sleep(20_000_000), g)[1])
        pen = penalty(m)
        torch.autograd.backward([act, pen], [dact, torch.ones_like(pen)])
    torch.cuda.synchronize()
    same(m, want)
    del kept


@pytest.mark.gpu
def test_a_capture_beside_an_older_graph_is_refused():
    m = build("cuda", 8).model.train()
    x = torch.randn(33, 5, device="cuda")
    kept = m(x)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(graph):
            x.add(1.0)
            m(x)
    del kept
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = m(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held.detach(), m(x).detach())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("train", [True, False])
def test_a_diverged_weight_shows(dev, bits, train):
    """A NaN that a block's Linear makes is a NaN behind the block's ReLU, as torch's is: in every row from that depth on, and in the gradients."""
    m = build(dev, bits).model.train(train)
    with torch.no_grad():
        m.stochstic_layers[1].block[0].weight[3, 7] = float("nan")
    x = torch.randn(33, 5, device=dev)
    act = m(x)
    assert torch.isfinite(act[:2]).all() and torch.isnan(act[2:]).all()
    if train and (dev == "cuda" or bits == 32):  # (the CPU stand-in's checkpoints read a group without numbers back as zeros)
        act.backward(torch.ones_like(act))
        for n, p in m.named_parameters():
            if not n.startswith("stochstic_layers.2") and n not in ("output_layer.bias", "stochstic_layers.1.block.2.bias"):
                assert torch.isnan(p.grad).any(), n
