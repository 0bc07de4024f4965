"""Block quantization, its inverse and the derivative form of an 8-bit checkpoint, against the numpy yardstick.

Bytes, scales and dz are compared for equality: the scales are powers of two, so every step before the one rounding to
e4m3 is exact (or, for dz, a fixed sequence of f32 roundings)."""
import ctypes

import numpy as np
import pytest

import _quant_ref as qr
import cleave_b200 as cb
from cleave_b200 import linalg, nn
from cleave_b200.linalg import QTensor, Tensor

pytestmark = pytest.mark.gpu
f32 = np.float32
FORMS = ["rows", "cols", "tiles"]
SIZES = [(1, 1), (1, 128), (1, 1024), (3, 17), (128, 128), (129, 257), (200, 1000), (1000, 3), (257, 516), (130, 4100)]

BIG = [(2300, 2100), (2177, 2511)]      # more tiles than are resident at once; 16-byte rows and others


def wide(rows, cols, seed=0):
    """Values whose magnitudes differ from row to row and column to column by many powers of two, zeros among them."""
    rng = np.random.default_rng(rows * 10007 + cols + seed)
    x = rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-12, 12, (rows, 1)) * 2.0 ** rng.integers(-6, 6, (1, cols))
    x[rng.random((rows, cols)) < 0.05] = 0.0
    return x.astype(f32)


def check_q(t: QTensor, want, cols):
    q, s = want
    assert np.array_equal(t.scales.numpy(), s)
    assert np.array_equal(t.numpy()[:, :cols], q[:, :cols])


def at_offset(a: np.ndarray, floats: int) -> Tensor:
    """The array in device memory `floats` elements behind an aligned address."""
    base = Tensor(np.concatenate([np.zeros(floats, f32), a.ravel()]))
    t = Tensor.from_device_ptr(base.data_ptr + 4 * floats, *a.shape)
    t._owner = base
    return t


@pytest.mark.parametrize("rows,cols", SIZES + BIG)
def test_quantize_every_form_alone_and_together(rows, cols):
    x = wide(rows, cols)
    want = {f: qr.quantize(x, f) for f in FORMS}
    t = Tensor(x)
    for f in FORMS:
        check_q(linalg.quantize(t, f), want[f], cols)
    for f, got in zip(FORMS, linalg.quantize(t, *FORMS)):
        check_q(got, want[f], cols)


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_quantize_reads_an_unaligned_tensor(offset):
    x = wide(150, 260, offset)
    t = at_offset(x, offset)
    for f, got in zip(FORMS, linalg.quantize(t, *FORMS)):
        check_q(got, qr.quantize(x, f), 260)


def test_quantize_edge_values():
    # block maxima at, just above and just below 1.75 * 2^k (where the scale steps), the type's extremes, subnormals, zeros
    top = f32(1.75)
    x = np.zeros((12, 128), f32)
    x[0, 5] = top
    x[1, 5] = np.nextafter(top, f32(2))
    x[2, 5] = np.nextafter(top, f32(0))
    x[3, :3] = [3.4028235e38, -1e30, 1e20]
    x[4, 7] = 1e-45
    x[5, :4] = [1e-38, -2e-39, 1e-40, 1e-45]
    x[6, 9] = 2.0 ** -126 * 448
    x[7, 9] = -448.0
    x[8, :4] = [-0.0, 0.0, -1.0, 2.0 ** -10]
    x[9, :4] = [448, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9]      # smallest subnormal, a tie to zero, a tie to even
    x[11, :] = np.arange(128) - 64
    for f in FORMS:
        check_q(linalg.quantize(Tensor(x), f), qr.quantize(x, f), 128)


def test_non_finite_values_become_nan_and_leave_their_block_alone():
    x = wide(130, 200)
    clean = x.copy()
    for r, c, v in ((0, 0, np.inf), (5, 130, -np.inf), (129, 199, np.nan), (64, 64, np.inf)):
        x[r, c], clean[r, c] = v, 0.0
    x[7, :128] = np.nan          # a whole block without a finite value
    clean[7, :128] = 0.0
    bad = ~np.isfinite(x)
    for f in FORMS:
        t = linalg.quantize(Tensor(x), f)
        q, s = qr.quantize(clean, f)
        got = t.numpy()[:, :200]
        assert np.array_equal(t.scales.numpy(), s)
        assert np.array_equal(got[~bad], q[:, :200][~bad])
        assert np.all((got[bad] & 0x7F) == 0x7F)


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("form", FORMS)
def test_dequantize_is_exact(rows, cols, form):
    x = wide(rows, cols, 1)
    t = linalg.quantize(Tensor(x), form)
    q, s = qr.quantize(x, form)
    want = qr.values(q, s, form, cols).astype(f32)
    assert np.array_equal(linalg.dequantize(t).numpy(), want)
    out = at_offset(np.full((rows, cols), 7, f32), 1)
    assert np.array_equal(linalg.dequantize(t, out).numpy(), want)


def test_uploaded_bytes_come_back_and_padding_is_never_read():
    q, s = qr.quantize(wide(40, 130), "cols")
    q[:, 130:] = 0x7F                                   # NaN in every padding byte
    t = QTensor.from_numpy(q, s, 130, "cols")
    assert np.array_equal(t.numpy(), q)
    want = qr.values(q, s, "cols", 130).astype(f32)
    assert np.array_equal(linalg.dequantize(t).numpy(), want)
    g = wide(40, 130, 2)
    outs = QTensor(40, 130, "rows"), QTensor(40, 130, "cols")
    nn.act_bwd_q(t, Tensor(g), "tanh", *outs)
    dz = qr.act_bwd_f32(want, g, "tanh")
    for o in outs:
        check_q(o, qr.quantize(dz, o.blocks), 130)


# ---- derivative form ---------------------------------------------------------------------------------------------------
ACT_F = {"tanh": np.tanh, "sigmoid": lambda z: 1 / (1 + np.exp(-z)), "relu": lambda z: np.maximum(z, 0), "identity": lambda z: z}


def checkpoint(rows, cols, act, form, seed=3):
    rng = np.random.default_rng(seed + rows + cols)
    y = ACT_F[act](rng.standard_normal((rows, cols))).astype(f32)
    q, s = qr.quantize(y, form)
    return QTensor.from_numpy(q, s, cols, form), qr.values(q, s, form, cols).astype(f32)


def assert_colsum(got, dz):
    # f32 sums over at most 16 + 8 values in a row of additions per 128-row block, then over the blocks: every addition is off
    # by at most 2^-24 of a partial sum, which sum |dz| bounds
    rows = dz.shape[0]
    blocks = -(-rows // 128)
    d64 = dz.astype(np.float64)
    bound = (24 + blocks) * 2.0 ** -24 * np.abs(d64).sum(0) + 1e-44
    assert np.all(np.abs(got.astype(np.float64) - d64.sum(0)) <= bound)


@pytest.mark.parametrize("rows,cols", SIZES + BIG)
@pytest.mark.parametrize("act", ["tanh", "sigmoid", "relu", "identity"])
def test_act_bwd_all_outputs(rows, cols, act):
    y, y_val = checkpoint(rows, cols, act, "cols")
    g = wide(rows, cols, 5) * f32(2.0 ** -18)
    dz, db = Tensor.empty(rows, cols), Tensor.empty(cols)
    outs = QTensor(rows, cols, "cols"), QTensor(rows, cols, "rows")
    nn.act_bwd_q(y, Tensor(g), act, *outs, dz=dz, db=db)
    want = qr.act_bwd_f32(y_val, g, act)
    assert np.array_equal(dz.numpy(), want)
    for o in outs:
        check_q(o, qr.quantize(want, o.blocks), cols)
    assert_colsum(db.numpy(), want)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("give", ["dz", "rows", "cols", "db"])
def test_act_bwd_each_output_alone_from_each_checkpoint_form(form, give):
    rows, cols = 300, 261
    y, y_val = checkpoint(rows, cols, "tanh", form)
    g = wide(rows, cols, 6)
    want = qr.act_bwd_f32(y_val, g, "tanh")
    tg = at_offset(g, 3)
    if give == "dz":
        dz = at_offset(np.zeros((rows, cols), f32), 1)
        nn.act_bwd_q(y, tg, "tanh", dz=dz)
        assert np.array_equal(dz.numpy(), want)
    elif give == "db":
        db = Tensor.empty(cols)
        nn.act_bwd_q(y, tg, "tanh", db=db)
        assert_colsum(db.numpy(), want)
    else:
        o = QTensor(rows, cols, give)
        nn.act_bwd_q(y, tg, "tanh", o)
        check_q(o, qr.quantize(want, give), cols)


@pytest.mark.parametrize("act", ["tanh", "sigmoid"])
def test_act_bwd_against_differences(act):
    # d act(z) * g by central differences in 64 bits.  The checkpoint's y is off by at most 2^-4 |y| (half an e4m3 step; y is
    # far above the block's subnormals here), so 1 - y^2 is off by at most 2^-3 y^2 + 2^-8 y^2 and y (1 - y) by at most
    # 2^-4 |y| |1 - 2 y| + 2^-8 y^2; the differences themselves by h^2 / 6 * max|act'''| < 1e-6 for h = 1e-3.
    rng = np.random.default_rng(11)
    z = rng.uniform(0.5, 2.0, (64, 128))
    g = rng.standard_normal((64, 128)).astype(f32)
    f, h = ACT_F[act], 1e-3
    slope = (f(z + h) - f(z - h)) / (2 * h)
    y = f(z)
    q, s = qr.quantize(y.astype(f32), "cols")
    dz = Tensor.empty(64, 128)
    nn.act_bwd_q(QTensor.from_numpy(q, s, 128, "cols"), Tensor(g), act, dz=dz)
    off = (2.0 ** -3 * y ** 2 if act == "tanh" else 2.0 ** -4 * y * np.abs(1 - 2 * y)) + 2.0 ** -8 * y ** 2 + 2e-6
    assert np.all(np.abs(dz.numpy() - slope * g) <= off * np.abs(g))


def test_relu_checkpoint_keeps_every_sign():
    # what relu's derivative needs of y is whether it is positive: values 2^10 below the block's maximum still are in 8 bits
    y = np.zeros((128, 4), f32)
    y[0] = 1.0
    y[1:5, 0] = [2.0 ** -10, 2.0 ** -17, 2.0 ** -18, 2.0 ** -30]
    t = linalg.quantize(Tensor(y), "cols")
    g = np.ones((128, 4), f32)
    dz = Tensor.empty(128, 4)
    nn.act_bwd_q(t, Tensor(g), "relu", dz=dz)
    # scale 2^-8 (1 <= 448 * 2^-8): the smallest e4m3 value is 2^-9 * 2^-8 = 2^-17; half of it ties to zero
    assert list(dz.numpy()[1:5, 0]) == [1.0, 1.0, 0.0, 0.0]


def test_captured_pass_replays_on_new_values():
    rows, cols = 260, 388
    y, y_val = checkpoint(rows, cols, "tanh", "cols")
    g1, g2 = wide(rows, cols, 7), wide(rows, cols, 8)
    tg = Tensor(g1)
    out, db = QTensor(rows, cols, "rows"), Tensor.empty(cols)
    graph = cb.StepGraph(lambda: nn.act_bwd_q(y, tg, "tanh", out, db=db))
    c_f32p = ctypes.POINTER(ctypes.c_float)
    for g in (g2, g1):
        assert cb.lib().cleave_cuda_upload_into_f32(tg._h, g.ctypes.data_as(c_f32p), g.size) == 0
        graph.replay()
        cb.sync()
        want = qr.act_bwd_f32(y_val, g, "tanh")
        check_q(out, qr.quantize(want, "rows"), cols)
        assert_colsum(db.numpy(), want)
    graph.close()


# ---- refusals ----------------------------------------------------------------------------------------------------------
def refused(code, call):
    L = cb.lib()
    assert call() == -code, L.cleave_cuda_last_error_message()
    assert L.cleave_cuda_last_error() == code
    L.cleave_cuda_clear_error()


def test_library_refuses_what_does_not_fit():
    L = cb.lib()
    x = Tensor(wide(64, 96))
    o = {f: QTensor(64, 96, f) for f in FORMS}
    h = {f: (t._h, t.scales._h) for f, t in o.items()}
    none = (None, None)
    refused(4, lambda: L.cleave_cuda_quantize_e4m3(x._h, 64, 96, *none, *none, *none))                  # no output
    refused(3, lambda: L.cleave_cuda_quantize_e4m3(x._h, 96, 64, *h["rows"], *none, *none))             # another shape
    refused(3, lambda: L.cleave_cuda_quantize_e4m3(x._h, 64, 95, *h["rows"], *none, *none))
    refused(2, lambda: L.cleave_cuda_quantize_e4m3(x._h, 64, 96, h["rows"][0], None, *none, *none))     # half an output
    refused(4, lambda: L.cleave_cuda_quantize_e4m3(x._h, 64, 96, x._h, h["rows"][1], *none, *none))     # f32 for bytes
    refused(4, lambda: L.cleave_cuda_quantize_e4m3(h["rows"][0], 64, 96, *h["rows"], *none, *none))     # bytes for f32
    refused(4, lambda: L.cleave_cuda_quantize_e4m3(x._h, 64, 96, h["rows"][0], h["rows"][1], h["rows"][0], h["cols"][1], *none))
    refused(4, lambda: L.cleave_cuda_dequantize_e4m3(x._h, *h["rows"], 64, 96, 4))                      # unknown form
    refused(3, lambda: L.cleave_cuda_dequantize_e4m3(x._h, *h["rows"], 64, 96, 2))                      # scales of another form
    refused(4, lambda: L.cleave_cuda_dequantize_e4m3(x._h, *h["rows"], 0, 96, 1))
    y, g = o["cols"], x
    z = Tensor.empty(64, 96)
    z_row = Tensor.from_device_ptr(z.data_ptr, 96)
    args = (*h["cols"], 2, g._h, 64, 96)
    refused(4, lambda: L.cleave_cuda_act_bwd_e4m3(*args, 3, None, *none, *none, None))                  # no output
    refused(4, lambda: L.cleave_cuda_act_bwd_e4m3(*args, 9, z._h, *none, *none, None))                  # unknown activation
    refused(4, lambda: L.cleave_cuda_act_bwd_e4m3(*args, 3, g._h, *none, *none, None))                  # in place
    refused(4, lambda: L.cleave_cuda_act_bwd_e4m3(*args, 3, None, *none, *h["cols"], None))             # over its own checkpoint
    refused(3, lambda: L.cleave_cuda_act_bwd_e4m3(*args, 3, None, *none, *none, z._h))                  # db of a matrix's length
    refused(4, lambda: L.cleave_cuda_act_bwd_e4m3(*args, 3, z._h, *none, *none, z_row._h))                # two outputs meet
    assert L.cleave_cuda_wrap_e4m3(ctypes.c_void_p(x.data_ptr + 4), 64) is None and L.cleave_cuda_last_error() == 4
    assert L.cleave_cuda_alloc_e4m3(0) is None
    L.cleave_cuda_clear_error()
    buf = np.zeros(64 * 96, f32)
    p = buf.ctypes.data_as(ctypes.POINTER(ctypes.c_float))
    refused(4, lambda: L.cleave_cuda_upload_async_f32(h["rows"][0], p, 64 * 96))                        # 4 bytes a byte
    refused(4, lambda: L.cleave_cuda_download_async_f32(h["rows"][0], p, 64 * 96))
    refused(4, lambda: L.cleave_cuda_upload_into_f32(h["rows"][0], p, 64 * 96))
    assert L.cleave_cuda_add_f32(h["rows"][0], h["rows"][0]) is None and L.cleave_cuda_last_error() == 4
    L.cleave_cuda_clear_error()
    cb.sync()
