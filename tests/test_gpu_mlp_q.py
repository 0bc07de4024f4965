"""A perceptron step with 8-bit products, stage by stage: every stage is compared with the same stage in 64 bits on the
values that the quantized operands stand for, taken from the device's own input of that stage."""
import numpy as np
import pytest

import _quant_ref as qr
import cleave_b200 as cb
from cleave_b200 import autodiff, linalg, workloads

pytestmark = pytest.mark.gpu
f32 = np.float32
SIZES = [(4, 3, 5, 2), (100, 130, 70, 33), (256, 128, 512, 64), (384, 200, 1000, 129)]


def deq(x, form):
    q, s = qr.quantize(x, form)
    return qr.values(q, s, form, x.shape[1])


def product_bound(a, b):
    """Error bound of the device's a @ b (see the product's tests)."""
    return (128 * 2 + 3 + -(-a.shape[1] // 128) + 8) * 2.0 ** -24 * (np.abs(a) @ np.abs(b))


def case(batch, d_in, d_hid, d_out):
    X, W1, _, W2, _, T = workloads.mlp_inputs(batch, d_in, d_hid, d_out)
    return X, W1, workloads.uniform_pm1(41, d_hid) * f32(0.1), W2, workloads.uniform_pm1(42, d_out) * f32(0.1), T


@pytest.mark.parametrize("batch,d_in,d_hid,d_out", SIZES)
def test_step_matches_64_bits_stage_by_stage(batch, d_in, d_hid, d_out):
    X, W1, b1, W2, b2, T = case(batch, d_in, d_hid, d_out)
    net = autodiff.MLP2(d_in, d_hid, d_out, products="e4m3")
    net.load(W1, b1, W2, b2)
    loss, inter = net.forward_backward(linalg.Tensor(X), linalg.Tensor(T), keep=True)
    v = {k: t.numpy() for k, t in inter.items()}
    Xr, Xc, W1q, W2q = deq(X, "rows"), deq(X, "cols"), deq(W1, "tiles"), deq(W2, "tiles")

    z = Xr @ W1q + b1
    assert np.all(np.abs(v["H"] - np.tanh(z)) <= product_bound(Xr, W1q) + 2.0 ** -24 * np.abs(z) + 4e-7)
    Hr, Hc = deq(v["H"], "rows"), deq(v["H"], "cols")
    z = Hr @ W2q + b2
    assert np.all(np.abs(v["Y"] - 1 / (1 + np.exp(-z))) <= product_bound(Hr, W2q) + 2.0 ** -24 * np.abs(z) + 4e-7)
    y = v["Y"].astype(np.float64)
    assert abs(loss - np.mean((y - T) ** 2)) <= 1e-5 * loss
    dz2 = 2 * (y - T) / y.size * y * (1 - y)
    assert np.all(np.abs(v["dZ2"] - dz2) <= 1e-5 * np.abs(dz2) + 2.0 ** -22 / y.size)      # y - T cancels
    dZr, dZc = deq(v["dZ2"], "rows"), deq(v["dZ2"], "cols")
    assert np.all(np.abs(v["dH"] - dZr @ W2q.T) <= product_bound(dZr, W2q.T))
    assert np.array_equal(v["dZ1"], qr.act_bwd_f32(Hc.astype(f32), v["dH"], "tanh"))
    dZ1c = deq(v["dZ1"], "cols")
    assert np.all(np.abs(net.dW1.numpy() - Xc.T @ dZ1c) <= product_bound(Xc.T, dZ1c))
    assert np.all(np.abs(net.dW2.numpy() - Hc.T @ dZc) <= product_bound(Hc.T, dZc))
    rows = -(-batch // 128) + 26 + batch // 64
    for db, dz in ((net.db1, v["dZ1"]), (net.db2, v["dZ2"])):
        d = dz.astype(np.float64)
        assert np.all(np.abs(db.numpy() - d.sum(0)) <= max(rows, 100) * 2.0 ** -24 * np.abs(d).sum(0))
    # without the intermediates, with the loss left on the device: the same bits
    kept = net.grads.numpy().copy()
    out = linalg.Tensor.zero(1)
    assert net.forward_backward(linalg.Tensor(X), linalg.Tensor(T), loss_out=out) is None
    cb.sync()
    assert out[0] == loss and np.array_equal(net.grads.numpy(), kept)
    H, Y = net.forward(linalg.Tensor(X))
    assert np.array_equal(H.numpy(), v["H"]) and np.array_equal(Y.numpy(), v["Y"])


def test_formula_of_the_step_against_differences():
    # the stages above, without quantization, are the derivative of the loss: checked against central differences in 64 bits
    X, W1, b1, W2, b2, T = (a.astype(np.float64) for a in case(20, 9, 13, 5))

    def loss(W1, b1, W2, b2):
        return np.mean((1 / (1 + np.exp(-(np.tanh(X @ W1 + b1) @ W2 + b2))) - T) ** 2)

    H = np.tanh(X @ W1 + b1)
    Y = 1 / (1 + np.exp(-(H @ W2 + b2)))
    dZ2 = 2 * (Y - T) / Y.size * Y * (1 - Y)
    dZ1 = (1 - H * H) * (dZ2 @ W2.T)
    grads = [X.T @ dZ1, dZ1.sum(0), H.T @ dZ2, dZ2.sum(0)]
    rng = np.random.default_rng(1)
    p = [W1, b1, W2, b2]
    for i, g in enumerate(grads):
        d = rng.standard_normal(g.shape)
        h = 1e-5
        up, down = [a + h * d if j == i else a for j, a in enumerate(p)], [a - h * d if j == i else a for j, a in enumerate(p)]
        assert abs((loss(*up) - loss(*down)) / (2 * h) - np.sum(g * d)) <= 1e-8


def test_captured_step_and_hooks():
    X, W1, b1, W2, b2, T = case(256, 128, 256, 128)
    net = autodiff.MLP2(128, 256, 128, products="e4m3")
    net.load(W1, b1, W2, b2)
    tX, tT, out = linalg.Tensor(X), linalg.Tensor(T), linalg.Tensor.zero(1)
    order = []
    net.forward_backward(tX, tT, loss_out=out, on_grads_ready=lambda i: order.append(("ready", i)),
                         before_layer=lambda i: order.append(("before", i)))
    assert order == [("before", 1), ("before", 2), ("ready", 1), ("ready", 0)]
    cb.sync()
    want_loss, want = out[0], net.grads.numpy().copy()
    g = cb.StepGraph(lambda: net.forward_backward(tX, tT, loss_out=out))
    for _ in range(2):
        linalg.Tensor.filled(3.0, net.n_params)
        g.replay()
        cb.sync()
        assert out[0] == want_loss and np.array_equal(net.grads.numpy(), want)
    g.close()


def test_unknown_products_are_refused():
    with pytest.raises(ValueError):
        autodiff.MLP2(4, 4, 4, products="e5m2")
