"""The LayerNorm trunk's host side on the CPU stand-in: staging, buffers, wrappers, sharding over gloo ranks."""
import contextlib
import io
import os

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from oracle import dun_oracle as O
from tests.test_distributed_cpu import _free_port, _record_collectives


@pytest.fixture(autouse=True)
def stand_in():
    from dun_amd import kernels
    from tests.cpu_rows import CpuRowBackend
    kernels.set_backend(CpuRowBackend())
    yield
    kernels.set_backend(None)


def build(din=5, outs=1, W=40, L=3, bits=32, vi=True, regression=True, N=300, seed=0, lr=1e-2):
    from dun_amd.probability import depth_categorical, depth_categorical_VI
    from dun_amd.stochastic_fc_models import arq_uncert_fc_resnet_ln
    from dun_amd.training_wrappers import DUN, DUN_VI
    torch.manual_seed(seed)
    prior = [1.0 / (L + 1)] * (L + 1)
    with contextlib.redirect_stdout(io.StringIO()):
        model = arq_uncert_fc_resnet_ln(din, outs, W, L, act_bits=bits)
        pm = (depth_categorical_VI if vi else depth_categorical)(prior, cuda=False)
        return (DUN_VI if vi else DUN)(model, pm, N, lr=lr, momentum=0.5, cuda=False, regression=regression)


def plain(model, x):
    """The same function from the modules themselves, recorded by autograd."""
    h = model.input_layer(x)
    out = [model.output_layer(h)]
    for blk in model.stochstic_layers:
        h = blk(h, 1.0)
        out.append(model.output_layer(h))
    return torch.stack(out)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("outs", [1, 4])
def test_forward_and_gradients(bits, outs):
    net = build(outs=outs, bits=bits)
    m = net.model.train()
    x = torch.randn(33, 5)
    dact = torch.randn(4, 33, outs)
    act = m(x)
    want = plain(m, x)
    assert torch.allclose(act, want, rtol=1e-4, atol=1e-5)
    act.backward(dact)
    got = m.flat_grads.clone()
    params = list(m.parameters())
    ref = torch.autograd.grad(want, params, dact)
    for p, r in zip(params, ref):
        scale = r.norm() + 1e-6
        assert (p.grad - r).norm() <= (1e-4 if bits == 32 else 0.05) * scale, p.shape
    assert torch.equal(got, m.flat_grads)


def test_a_batch_of_one_row_trains_and_prediction_is_the_same_function():
    net = build()
    x, y = torch.randn(1, 5), torch.randn(1, 1)
    assert np.isfinite(net.fit(x, y)).all()
    x = torch.randn(7, 5)
    net.model.train()
    a = net.model(x).detach()
    net.model.eval()
    # (the head's sums of 40 products run in another order: off by at most 2 * 40 u sum |h w|, about 40 u * 2 * 20)
    same = lambda s, t: torch.allclose(s, t, rtol=0, atol=80 * 2.0 ** -24 * 20)
    assert same(a, net.model(x)) and net.predict(x).shape == (7, 1)
    assert torch.equal(net.predict(x, depth=3), net.predict(x))
    assert net.model(x, depth=1).shape == (2, 7, 1) and same(net.model(x, depth=1), a[:2])
    assert net.model(torch.empty(0, 5)).shape == (4, 0, 1)


def test_truncated_training_forward_leaves_no_stale_gradients():
    m = build().model.train()
    x = torch.randn(9, 5)
    m(x).sum().backward()
    act = m(x, depth=1)
    act.backward(torch.ones_like(act))
    want = torch.autograd.grad(plain(m, x)[:2].sum(), list(m.parameters()), allow_unused=True)
    for p, r in zip(m.parameters(), want):
        assert torch.allclose(p.grad, torch.zeros_like(p) if r is None else r, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoints_and_pickles(tmp_path, bits):
    net = build(bits=bits)
    x, y = torch.randn(20, 5), torch.randn(20, 1)
    net.fit(x, y)
    with contextlib.redirect_stdout(io.StringIO()):
        net.save_state(str(tmp_path / "s.pt"))
        net.save(str(tmp_path / "s.dat"))
        a, b = build(bits=bits, seed=1), build(bits=bits, seed=2)
        a.load_state(str(tmp_path / "s.pt"))
        b.load(str(tmp_path / "s.dat"))
    want = net.fit(x, y)
    assert a.fit(x, y) == want and b.fit(x, y) == want
    assert torch.equal(a.model.flat_params, net.model.flat_params) and b.model.act_bits == bits


def test_refusals():
    from dun_amd.stochastic_fc_models import arq_uncert_fc_resnet_ln
    with pytest.raises(ValueError, match="act_bits"):
        arq_uncert_fc_resnet_ln(5, 1, 8, 2, act_bits=16)
    m = build().model.train()
    with pytest.raises(RuntimeError, match="expected x"):
        m(torch.randn(3, 4))
    with pytest.raises(RuntimeError, match="empty batch"):
        m(torch.empty(0, 5))
    act = m(torch.randn(3, 5))
    m(torch.randn(3, 5))
    with pytest.raises(RuntimeError, match="reused by a later"):
        act.sum().backward()


def test_keys_of_the_state_dict():
    m = build(L=1).model
    assert sorted(m.state_dict()) == ["input_layer.bias", "input_layer.weight", "output_layer.bias", "output_layer.weight",
                                      "stochstic_layers.0.block.0.bias", "stochstic_layers.0.block.0.weight",
                                      "stochstic_layers.0.block.2.bias", "stochstic_layers.0.block.2.weight"]


def _data(B, din=5):
    return O.synthetic_regression(B, din, seed=3)


def _rank(rank, world, port, bits, vi, buckets, ret):
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    torch.set_num_threads(2)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    log = []
    _record_collectives(log)
    try:
        from dun_amd import kernels
        from dun_amd.distributed import shard
        from tests.cpu_rows import CpuRowBackend
        kernels.set_backend(CpuRowBackend())
        net = build(bits=bits, vi=vi)
        if rank:
            net.model.flat_params.add_(0.5)
        with contextlib.redirect_stdout(io.StringIO()):
            shard(net, grad_bucket_blocks=buckets)
        x, y = _data(48)
        B = 48 // world
        out = [net.fit(x[rank * B:(rank + 1) * B], y[rank * B:(rank + 1) * B]) for _ in range(3)]
        ret[rank] = (out, net.model.flat_params.numpy().copy(), log)
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("bits,vi,buckets,world", [(32, True, 2, 2), (8, True, 1, 2), (32, False, 5, 3)])
def test_ranks_match_a_single_process(bits, vi, buckets, world):
    ret = mp.Manager().dict()
    mp.spawn(_rank, args=(world, _free_port(), bits, vi, buckets, ret), nprocs=world, join=True)
    net = build(bits=bits, vi=vi)
    x, y = _data(48)
    want = [net.fit(x, y) for _ in range(3)]
    flat = net.model.flat_params.numpy()
    for r in range(world):
        assert np.allclose(ret[r][0], want, rtol=2e-5, atol=1e-6)
        assert np.array_equal(ret[r][1], ret[0][1]) and ret[r][2] == ret[0][2]
        assert np.abs(ret[r][1] - flat).max() <= 2e-5 * np.abs(flat).max()
    # no statistics of a batch travel: one message of likelihood sums, one of metrics per step, and gradients
    small = [m for m in ret[0][2] if m[0] == "all_reduce" and m[2] == "torch.float64"]
    assert all(m[1] in ((4,), (2,)) for m in small), small
