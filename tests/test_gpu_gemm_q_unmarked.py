"""A tensor whose scales are not powers of two and that is not marked so: the large product, which reads exponents only, reports it."""
import numpy as np
import pytest

import cleave_b200 as cb
from cleave_b200 import linalg
from cleave_b200.linalg import QTensor, Tensor
from test_gpu_gemm_q_long import operand

pytestmark = pytest.mark.gpu
f32 = np.float32
M, N, K = 1300, 1281, 700


def with_scale(t, at, value):
    s = t.scales.numpy().copy()
    s[at] = value
    u = QTensor.from_numpy(t.numpy(), s, t.dims[1], t.blocks)
    assert u.any_scales
    return u


def unmarked(t):
    t.any_scales, t.form = False, linalg.BLOCKS[t.blocks]
    return t


@pytest.mark.parametrize("value", [1.5, -1.0, 0.0, np.inf, np.nan, 2.0 ** -127, 2.0 ** -149, np.nextafter(f32(1), f32(2))])
@pytest.mark.parametrize("at", [(0, 0), (-1, -1), (3, 130)])
def test_large_product_reports_it(value, at):
    a, _ = operand(1, M, K, False, "rows")
    b, _ = operand(2, N, K, True, "tiles")
    c = Tensor.empty(M, N)
    odd = unmarked(with_scale(a, at, value))
    linalg.gemm_q_into(c, odd, b)
    with pytest.raises(cb.CleaveCudaError, match="first operand") as e:
        c.numpy()
    assert e.value.code == 4
    odd = unmarked(with_scale(b, (at[0], at[1] % b.scale_dims[1]), value))
    linalg.gemm_q_into(c, a, odd)
    assert cb.lib().cleave_cuda_sync() == 4
    assert b"second operand" in cb.lib().cleave_cuda_last_error_message()
    cb.lib().cleave_cuda_clear_error()
    # the report is given once, and the next product is right
    good = linalg.gemm_q_into(c, a, b).numpy()
    assert np.array_equal(good, linalg.gemm_q_into(Tensor.empty(M, N), a, b).numpy())


def test_ends_of_the_range_are_powers_of_two():
    a, _ = operand(1, M, K, False, "rows")
    b, _ = operand(2, N, K, True, "tiles")
    s = a.scales.numpy().copy()
    s[0, 0], s[-1, -1] = 2.0 ** -126, 2.0 ** 127
    u = QTensor.from_numpy(a.numpy(), s, K, "rows")
    assert not u.any_scales
    linalg.gemm_q_into(Tensor.empty(M, N), u, b)
    assert cb.lib().cleave_cuda_sync() == 0


def test_small_products_take_the_scales_as_they_are():
    a, _ = operand(1, 100, K, False, "rows")
    b, _ = operand(2, N, K, True, "tiles")
    odd = with_scale(a, (3, 30), 1.5)
    want = linalg.gemm_q_into(Tensor.empty(100, N), odd, b).numpy()
    assert np.array_equal(linalg.gemm_q_into(Tensor.empty(100, N), unmarked(odd), b).numpy(), want)
