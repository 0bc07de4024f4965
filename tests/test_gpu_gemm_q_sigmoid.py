"""The sigmoid of the 8-bit product's epilogue over its whole range, relative to its value.

The sum is one exact product (a value of A times 1), so the result is the sigmoid's alone: an exponential and a
reciprocal within 2^-23, a sum and a product within 2^-24: 3.6e-7 in all, below 4e-7.  Results under 2^-126 have a step of 2^-149."""
import numpy as np
import pytest

import _quant_ref as qr
from cleave_b200 import linalg
from cleave_b200.linalg import QTensor, Tensor

pytestmark = pytest.mark.gpu
f32 = np.float32


def one_column(v, scale):
    """v / scale (e4m3 values) as an 8-bit tensor [len(v), 1]."""
    q = np.zeros((v.size, 16), np.uint8)
    q[:, 0] = qr.encode(v / scale)
    return QTensor.from_numpy(q, np.full((1, v.size), scale, f32), 1, "rows")


@pytest.mark.parametrize("repeat", [1, 24])   # few rows: one CTA a tile; many: CTA pairs
@pytest.mark.parametrize("n", [4, 1281])
def test_relative_error_of_the_sigmoid(repeat, n):
    values = np.tile(np.array([s * m * 2.0 ** e for s in (1, -1) for e in range(-3, 5) for m in range(8, 16)]), repeat)   # -240 .. 240
    a = one_column(values, 1.0)
    b = QTensor.from_numpy(np.full((n, 16), qr.encode(np.ones(1))[0], np.uint8), np.ones((1, n), f32), 1, "rows")
    bias = np.where(np.arange(n) % 2 == 0, 0.0, 0.125).astype(f32)
    c = linalg.gemm_q_into(Tensor.filled(np.nan, values.size, n), a, b, trans_b=True, bias=Tensor(bias), act="sigmoid").numpy()
    z = (values[:, None].astype(f32) + bias[None, :]).astype(np.float64)
    want = np.where(z < 0, np.exp(np.minimum(z, 0)) / (1 + np.exp(np.minimum(z, 0))), 1 / (1 + np.exp(-np.maximum(z, 0))))
    off = np.abs(c - want) - 4e-7 * want
    assert np.all(off <= 2.0 ** -149), (float(off.max()), float(z.reshape(-1)[np.argmax(off)]))
