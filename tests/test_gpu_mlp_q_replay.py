"""The perceptron's 8-bit step replayed and repeated, with every output overwritten before it is written again, and at sizes whose
products take CTA pairs."""
import numpy as np
import pytest

import cleave_b200 as cb
import test_gpu_mlp_q as steps
from cleave_b200 import autodiff, linalg, nn
from cleave_b200._lib import c_f32p

pytestmark = pytest.mark.gpu
f32 = np.float32


def overwrite(t, a):
    a = np.ascontiguousarray(a, f32)
    assert cb.lib().cleave_cuda_upload_into_f32(t._h, a.ctypes.data_as(c_f32p), a.size) == 0
    cb.sync()


def wipe(net, out):
    overwrite(net.grads, np.full(net.n_params, np.nan))
    overwrite(out, [np.nan])


@pytest.mark.parametrize("batch,d_in,d_hid,d_out", [(256, 128, 256, 128), (100, 130, 70, 33), (1300, 640, 1300, 640)])
def test_replays_write_everything_and_read_the_new_batch(batch, d_in, d_hid, d_out):
    X, W1, b1, W2, b2, T = steps.case(batch, d_in, d_hid, d_out)
    other = (X[::-1] * f32(1.5), T[::-1])
    net = autodiff.MLP2(d_in, d_hid, d_out, products="e4m3")
    net.load(W1, b1, W2, b2)
    tX, tT, out = linalg.Tensor(X), linalg.Tensor(T), linalg.Tensor.zero(1)
    want = []
    for x, t in ((X, T), other):
        overwrite(tX, x)
        overwrite(tT, t)
        wipe(net, out)
        loss, inter = net.forward_backward(tX, tT, keep=True)
        kept = net.grads.numpy().copy()
        assert np.isfinite(kept).all()
        wipe(net, out)      # without the intermediates: the same gradients, written anew
        net.forward_backward(tX, tT, loss_out=out)
        cb.sync()
        assert out[0] == loss and np.array_equal(net.grads.numpy(), kept)
        want.append((loss, kept))
    assert not np.array_equal(want[0][1], want[1][1])
    g = cb.StepGraph(lambda: net.forward_backward(tX, tT, loss_out=out))
    for i in (0, 1, 0):
        x, t = ((X, T), other)[i]
        overwrite(tX, x)
        overwrite(tT, t)
        wipe(net, out)
        scratch = [linalg.Tensor(np.full(batch * d_hid, np.nan, f32)) for _ in range(3)]   # blocks that no replay may be using
        g.replay()
        cb.sync()
        assert out[0] == want[i][0] and np.array_equal(net.grads.numpy(), want[i][1])
        assert all(np.isnan(s.numpy()).all() for s in scratch)
    # new weights reach a replay as well
    overwrite(net.params, net.params.numpy() * f32(0.5))
    wipe(net, out)
    net.forward_backward(tX, tT, loss_out=out)
    cb.sync()
    loss, grads = out[0], net.grads.numpy().copy()
    wipe(net, out)
    g.replay()
    cb.sync()
    assert out[0] == loss and np.array_equal(net.grads.numpy(), grads)
    g.close()


def test_two_captured_steps_do_not_share_what_they_write():
    cases = [steps.case(256, 128, 256, 128), steps.case(300, 70, 300, 40)]
    nets, graphs, want = [], [], []
    for X, W1, b1, W2, b2, T in cases:
        net = autodiff.MLP2(X.shape[1], W1.shape[1], T.shape[1], products="e4m3")
        net.load(W1, b1, W2, b2)
        tX, tT, out = linalg.Tensor(X), linalg.Tensor(T), linalg.Tensor.zero(1)
        net.forward_backward(tX, tT, loss_out=out)
        cb.sync()
        want.append((out[0], net.grads.numpy().copy()))
        graphs.append(cb.StepGraph(lambda net=net, tX=tX, tT=tT, out=out: net.forward_backward(tX, tT, loss_out=out)))
        nets.append((net, out, tX, tT))
    for net, out, *_ in nets:
        wipe(net, out)
    for _ in range(3):
        for g in graphs:
            g.replay()
    cb.sync()
    for (net, out, *_), (loss, grads) in zip(nets, want):
        assert out[0] == loss and np.array_equal(net.grads.numpy(), grads)
    for g in graphs:
        g.close()


def test_step_on_cta_pairs_matches_64_bits_stage_by_stage():
    # every product has 24 to 64 tiles of 256 x 256, contractions of 640 to 2048, bias, tanh and sigmoid
    steps.test_step_matches_64_bits_stage_by_stage(2048, 640, 2048, 640)


def test_checkpoint_backward_in_a_graph_with_many_row_blocks():
    # column sums over row blocks by the last CTA (300 rows) and by a kernel of their own (17000 rows), replayed
    for rows in (300, 17000):
        rng = np.random.default_rng(rows)
        y, gr = linalg.Tensor(rng.uniform(-1, 1, (rows, 130)).astype(f32)), linalg.Tensor(rng.standard_normal((rows, 130)).astype(f32))
        yq = linalg.quantize(y, "cols")
        dz, db = linalg.Tensor.zero(rows, 130), linalg.Tensor.zero(130)
        nn.act_bwd_q(yq, gr, "tanh", dz=dz, db=db)
        want = dz.numpy().copy(), db.numpy().copy()
        g = cb.StepGraph(lambda: nn.act_bwd_q(yq, gr, "tanh", dz=dz, db=db))
        for _ in range(3):
            overwrite(dz, np.full((rows, 130), np.nan))
            overwrite(db, np.full(130, np.nan))
            g.replay()
            cb.sync()
            assert np.array_equal(dz.numpy(), want[0]) and np.array_equal(db.numpy(), want[1])
        g.close()
