"""What the perceptron's 8-bit step keeps between its passes: the forms that the backward pass reads, and no others.

The step runs on stand-ins that compute nothing; each product notes which 8-bit tensors are alive when it is queued."""
import gc
import weakref

import pytest

from cleave_b200 import autodiff


class Fake:
    def __init__(self, name, *dims):
        self.name, self.dims = name, dims

    @staticmethod
    def empty(*dims):
        return Fake("f32", *dims)


@pytest.fixture
def step(monkeypatch):
    live, products = [], []

    def quantize(x, *forms):
        outs = tuple(Fake(f"{x.name} {f}", *x.dims) for f in forms)
        live.extend(weakref.ref(o) for o in outs)
        return outs if len(outs) > 1 else outs[0]

    def gemm(c, a, b, **how):
        gc.collect()
        products.append((a.name, b.name, {r().name for r in live if r() is not None}))
        c.name = {1: "H", 2: "Y", 3: "dH"}.get(len(products), c.name)
        return c

    def q_tensor(rows, cols, blocks):
        t = Fake("dZ1 " + blocks, rows, cols)
        live.append(weakref.ref(t))
        return t

    monkeypatch.setattr(autodiff, "quantize", quantize)
    monkeypatch.setattr(autodiff, "gemm_q_into", gemm)
    monkeypatch.setattr(autodiff, "QTensor", q_tensor)
    monkeypatch.setattr(autodiff, "Tensor", Fake)
    monkeypatch.setattr(autodiff.nn, "mse_act_bwd", lambda Y, T, act, out: (0.5, Fake("dZ2", *Y.dims)))
    monkeypatch.setattr(autodiff.nn, "act_bwd_q", lambda *a, **k: None)
    monkeypatch.setattr(autodiff.nn, "colsum_into", lambda *a: None)
    net = object.__new__(autodiff.MLP2)
    net.products, net.act1, net.act2, net.d_in, net.d_hid, net.d_out = "e4m3", "tanh", "sigmoid", 6, 7, 5
    for name, dims in (("W1", (6, 7)), ("b1", (7,)), ("W2", (7, 5)), ("b2", (5,)), ("dW1", (6, 7)), ("db1", (7,)), ("dW2", (7, 5)), ("db2", (5,))):
        setattr(net, name, Fake(name, *dims))
    return net, products


@pytest.mark.parametrize("keep", [False, True])
def test_row_forms_go_with_the_product_that_reads_them(step, keep):
    net, products = step
    net.forward_backward(Fake("X", 9, 6), Fake("T", 9, 5), keep=keep)
    assert [p[:2] for p in products] == [("X rows", "W1 tiles"), ("H rows", "W2 tiles"), ("dZ2 rows", "W2 tiles"), ("X cols", "dZ1 cols"),
                                         ("H cols", "dZ2 cols")]
    alive = [p[2] for p in products]
    assert alive[0] == {"X rows", "X cols", "W1 tiles"}
    assert alive[1] == {"X cols", "H rows", "H cols", "W2 tiles"}
    assert alive[2] == {"X cols", "H cols", "dZ2 rows", "dZ2 cols", "W2 tiles"}
    assert alive[3] == {"X cols", "H cols", "dZ1 cols", "dZ2 cols"}
    assert alive[4] == {"H cols", "dZ2 cols"}
