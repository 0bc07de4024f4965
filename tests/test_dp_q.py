"""Data-parallel training with 8-bit products: what the drivers allocate, and that a rank's step is the network's own."""
import types

import numpy as np
import pytest

import cleave_b200 as cb
from cleave_b200 import autodiff, dp, linalg, workloads


def test_lo_planes_only_for_products_that_read_them(monkeypatch):
    made = []
    monkeypatch.setattr(linalg, "Tensor", types.SimpleNamespace(empty=lambda *dims: made.append(dims) or dims))
    w = dict(W1=types.SimpleNamespace(dims=(6, 7)), W2=types.SimpleNamespace(dims=(7, 5)))
    assert dp._lo_planes(types.SimpleNamespace(products="e4m3", **w), 2) is None
    assert dp._lo_planes(types.SimpleNamespace(products="f32", **w), 1) is None and made == []
    assert dp._lo_planes(types.SimpleNamespace(products="f32", **w), 2) == [(7, 5), (6, 7)]
    assert dp._lo_planes(types.SimpleNamespace(**w), 2) == [(7, 5), (6, 7)]     # another replica class: as before


@pytest.fixture
def one_rank():
    import torch.distributed as dist
    dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    yield
    dist.destroy_process_group()


def problem(batch):
    X, W1, _, W2, _, T = workloads.mlp_inputs(batch, 64, 256, 32)
    b1, b2 = workloads.uniform_pm1(41, 256) * np.float32(0.1), workloads.uniform_pm1(42, 32) * np.float32(0.1)
    return X, T, (W1, b1, W2, b2)


@pytest.mark.gpu
def test_driver_of_one_rank_trains_as_the_network_does(one_rank):
    X, T, weights = problem(512)
    tX, tT = linalg.Tensor(X), linalg.Tensor(T)
    mine, theirs = (autodiff.MLP2(64, 256, 32, products="e4m3") for _ in range(2))
    for net in (mine, theirs):
        net.load(*weights)
    trainer = dp.DataParallel(dp.MLP2Replica(theirs))
    for _ in range(4):
        want = mine.forward_backward(tX, tT)
        mine.sgd(0.5, 1.0)
        assert trainer.step(tX, tT, 0.5) == want
    cb.sync()
    assert np.array_equal(theirs.params.numpy(), mine.params.numpy())


@pytest.mark.gpu
def test_mean_of_two_shards_is_the_gradient_of_the_batch():
    # shards of whole 128-row blocks quantize alike, the loss's 1/batch is a power of two, and at these sizes the products that run
    # along the batch take the same path for either number of rows: what is left is the order of the weight gradients' sums
    X, T, weights = problem(512)
    net = autodiff.MLP2(64, 256, 32, products="e4m3")
    net.load(*weights)
    net.forward_backward(linalg.Tensor(X), linalg.Tensor(T))
    whole = net.grads.numpy().astype(np.float64)
    shards = []
    for at in (slice(0, 256), slice(256, 512)):
        net.forward_backward(linalg.Tensor(np.ascontiguousarray(X[at])), linalg.Tensor(np.ascontiguousarray(T[at])))
        shards.append(net.grads.numpy().astype(np.float64))
    # each side is within (128 * 2 + 3 + 4 + 8) * 2^-24 of the sum of magnitudes; four of those cover both sides, and no gradient
    # here has magnitudes above 64 times its largest element
    assert np.all(np.abs(whole - (shards[0] + shards[1]) / 2) <= 4 * 271 * 2.0 ** -24 * 64 * np.abs(whole).max())
