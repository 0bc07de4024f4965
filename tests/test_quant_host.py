"""Host side of the 8-bit tensors: sizes, and what is refused before any device work."""
import numpy as np
import pytest

import cleave_b200 as cb
from cleave_b200 import autodiff, linalg, nn
from cleave_b200.linalg import QTensor, Tensor


def fake(*dims, dtype="f32"):
    return Tensor(dims=dims, dtype=dtype, _handle=0)     # a handle the library has never issued


def fake_q(rows, cols, blocks, any_scales=False):
    return QTensor(rows, cols, blocks, any_scales=any_scales, _handle=0, _scales=fake(1))


@pytest.mark.parametrize("rows,cols,pitch", [(1, 1, 16), (3, 16, 16), (3, 17, 32), (200, 1000, 1008), (2 ** 31 - 1, 1, 16)])
def test_sizes(rows, cols, pitch):
    L = cb.lib()
    rb, c = -(-rows // 128), -(-cols // 128)
    assert L.cleave_cuda_e4m3_bytes(rows, cols) == rows * pitch
    assert [L.cleave_cuda_e4m3_scales(rows, cols, b) for b in (1, 2, 3)] == [c * rows, rb * cols, rb * c]
    for b, dims in (("rows", (c, rows)), ("cols", (rb, cols)), ("tiles", (rb, c))):
        q = fake_q(rows, cols, b)
        assert q.nbytes == rows * pitch and q.scale_dims == dims
    assert L.cleave_cuda_e4m3_bytes(0, 5) == 0 and L.cleave_cuda_e4m3_scales(5, -1, 1) == 0
    assert L.cleave_cuda_e4m3_scales(rows, cols, 0) == 0 and L.cleave_cuda_e4m3_scales(rows, cols, 4) == 0


def test_block_form_of_the_c_abi():
    assert [fake_q(2, 2, b).form for b in ("rows", "cols", "tiles")] == [1, 2, 3]
    assert fake_q(2, 2, "cols", any_scales=True).form == 18


def test_shapes_and_forms_are_checked_like_type_errors():
    for bad in (lambda: QTensor(0, 4, "rows"), lambda: QTensor(4, -1, "rows"), lambda: QTensor(4, 4, "row"),
                lambda: QTensor(2 ** 31, 4, "rows"), lambda: QTensor.from_numpy(np.zeros((4, 8), np.uint8), np.ones((1, 4)), 8, "rows"),
                lambda: QTensor.from_numpy(np.zeros((4, 16), np.uint8), np.ones((4, 1)), 8, "rows"),
                lambda: QTensor.from_numpy(np.zeros(64, np.uint8), np.ones((1, 4)), 16, "rows")):
        with pytest.raises(TypeError):
            bad()
    x, rows, cols = fake(8, 20), fake_q(8, 20, "rows"), fake_q(8, 20, "cols")
    for bad in (lambda: linalg.quantize_into(x), lambda: linalg.quantize_into(x, fake_q(20, 8, "rows")),
                lambda: linalg.quantize_into(x, rows, fake_q(8, 20, "rows")), lambda: linalg.quantize_into(fake(160), rows),
                lambda: linalg.quantize_into(fake(8, 20, dtype="f64"), rows), lambda: linalg.quantize_into(x, fake(8, 20)),
                lambda: linalg.quantize(fake(4)), lambda: linalg.dequantize(rows, fake(20, 8)),
                lambda: linalg.dequantize(rows, fake(8, 20, dtype="f64"))):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: nn.act_bwd_q(cols, x, "tanh"), lambda: nn.act_bwd_q(cols, fake(20, 8), "tanh", rows),
                lambda: nn.act_bwd_q(x, x, "tanh", rows), lambda: nn.act_bwd_q(cols, x, "gelu", rows),
                lambda: nn.act_bwd_q(cols, x, "tanh", fake_q(8, 20, "tiles")), lambda: nn.act_bwd_q(cols, x, "tanh", dz=fake(160)),
                lambda: nn.act_bwd_q(cols, x, "tanh", rows, db=fake(8)), lambda: nn.act_bwd_q(cols, x, "tanh", rows, rows)):
        with pytest.raises(TypeError):
            bad()


def test_products_need_blocks_along_the_contraction():
    c = fake(8, 12)
    a, b = {f: fake_q(8, 20, f) for f in ("rows", "cols", "tiles")}, {f: fake_q(20, 12, f) for f in ("rows", "cols", "tiles")}
    for fa, fb in (("cols", "tiles"), ("rows", "rows"), ("tiles", "rows")):
        with pytest.raises(TypeError):
            linalg.gemm_q_into(c, a[fa], b[fb])
    for bad in (lambda: linalg.gemm_q_into(c, a["rows"], b["cols"], trans_b=True), lambda: linalg.gemm_q_into(fake(12, 8), a["rows"], b["cols"]),
                lambda: linalg.gemm_q_into(c, fake(8, 20), b["cols"]), lambda: linalg.gemm_q_into(c, a["rows"], b["cols"], bias=fake(8)),
                lambda: linalg.gemm_q_into(fake(8, 8), a["rows"], fake_q(8, 20, "cols"), trans_b=True)):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(ValueError):
        autodiff.MLP2(4, 4, 4, products="int8")


def test_entry_points_fail_loudly_without_live_handles():
    L = cb.lib()
    none = (None,) * 6
    for call in (lambda: L.cleave_cuda_quantize_e4m3(None, 4, 4, *none), lambda: L.cleave_cuda_dequantize_e4m3(None, None, None, 4, 4, 1),
                 lambda: L.cleave_cuda_gemm_e4m3(None, None, None, 1, None, None, 2, 4, 4, 4, 0, 0, None, 0),
                 lambda: L.cleave_cuda_act_bwd_e4m3(None, None, 2, None, 4, 4, 3, *none)):
        assert call() in (-1, -2)      # no device here; with one, no live handle
        assert L.cleave_cuda_last_error() in (1, 2)
        L.cleave_cuda_clear_error()
