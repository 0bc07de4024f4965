"""The block-scaled 8-bit product against 64-bit products of the values the operands stand for.

Error bound of an element, with S = sum over k of |a| |b| (the values).  The tensor pipe adds 32 exact products at a time into
an f32 accumulator that truncates, so at most 2^-23 of a partial sum per term summed there; it runs over at most 1024 terms
(eight k-blocks; one where the kernel scales them itself) before it is added to a running sum.  Taking every one of a k-block's
128 terms as an add of its own, as if it were the worst of them, covers the 32 adds of 1024 terms four times over: 128 * 2^-23 of
S.  Where the kernel scales, the scales' product and its product with the block's sum round three times, 3 * 2^-24; the
running sum adds at most 2^-24 of S per k-block and per rank of a split.  Together (128 * 2 + 3 + blocks + 8) * 2^-24 * S.  The
bias adds 2^-24 of the result, an activation is a contraction (slope at most 1) evaluated to within 4e-7 of its value."""
import ctypes

import numpy as np
import pytest

import _quant_ref as qr
import cleave_b200 as cb
from cleave_b200 import linalg
from cleave_b200.linalg import QTensor, Tensor

pytestmark = pytest.mark.gpu
f32 = np.float32
SIZES = [(1, 1, 1), (1, 128, 128), (3, 5, 7), (1, 700, 1024), (16, 16, 16), (17, 130, 129), (33, 257, 100), (64, 512, 384),
         (48, 300, 260), (65, 129, 640), (128, 128, 128), (129, 300, 513), (300, 40, 1000), (500, 9, 77), (256, 512, 2048),
         (257, 1031, 391)]
TRANS = [(0, 0), (0, 1), (1, 0), (1, 1)]


def operand(seed, free, k, stored_k_first, form):
    """An 8-bit operand with extent `free` and contraction length k, and its values as [free, k]."""
    rng = np.random.default_rng(seed)
    shape = (k, free) if stored_k_first else (free, k)
    x = rng.standard_normal(shape) * 2.0 ** rng.integers(-4, 4, (shape[0], 1)) * 2.0 ** rng.integers(-4, 4, (1, shape[1]))
    q, s = qr.quantize(x.astype(f32), form)
    q[:, shape[1]:] = 0x7F          # padding bytes are never read
    v = qr.values(q, s, form, shape[1])
    return QTensor.from_numpy(q, s, shape[1], form), (v.T if stored_k_first else v)


def forms(ta, tb):
    return [("cols" if ta else "rows", "tiles"), ("cols" if ta else "rows", "rows" if tb else "cols"), ("tiles", "tiles"),
            ("tiles", "rows" if tb else "cols")]


def bound(av, bv):
    blocks = -(-av.shape[1] // 128)
    return (128 * 2 + 3 + blocks + 8) * 2.0 ** -24 * (np.abs(av) @ np.abs(bv).T)


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("ta,tb", TRANS)
def test_product_every_order_and_block_form(m, n, k, ta, tb):
    for i, (fa, fb) in enumerate(forms(ta, tb)):
        a, av = operand(1 + i, m, k, ta, fa)
        b, bv = operand(50 + i, n, k, not tb, fb)
        c = linalg.gemm_q_into(Tensor.filled(np.nan, m, n), a, b, trans_a=bool(ta), trans_b=bool(tb)).numpy()
        err = np.abs(c.astype(np.float64) - av @ bv.T)
        assert np.all(err <= bound(av, bv)), (fa, fb, float(np.max(err / bound(av, bv))))


@pytest.mark.parametrize("m,n,k", [(1537, 1799, 391), (2048, 1284, 1024), (130, 9000, 128)])
@pytest.mark.parametrize("ta,tb", TRANS)
def test_large_product_every_order(m, n, k, ta, tb):
    # enough 256 x 256 tiles for CTA pairs; ragged edges, a width that TMA stores can take and one that they cannot
    for i, (fa, fb) in enumerate(forms(ta, tb)[:2]):
        a, av = operand(31 + i, m, k, ta, fa)
        b, bv = operand(41 + i, n, k, not tb, fb)
        bias = np.random.default_rng(5).standard_normal(n).astype(f32)
        c = linalg.gemm_q_into(Tensor.filled(np.nan, m, n), a, b, trans_a=bool(ta), trans_b=bool(tb), bias=Tensor(bias),
                               act="relu").numpy()
        z = av @ bv.T + bias
        assert np.all(np.abs(c - np.maximum(z, 0)) <= bound(av, bv) + 2.0 ** -24 * np.abs(z))


@pytest.mark.parametrize("m,n,k", [(1, 200, 300), (40, 333, 512), (150, 270, 1100), (513, 514, 515), (1700, 1600, 260)])
@pytest.mark.parametrize("ta,tb", TRANS)
def test_small_integers_are_exact(m, n, k, ta, tb):
    # integers up to 8 are e4m3 values, every partial sum is an integer below 2^24: no rounding anywhere
    rng = np.random.default_rng(m + n + k)
    ai, bi = rng.integers(-8, 9, (m, k)), rng.integers(-8, 9, (n, k))

    def q(v, stored_k_first, form):
        v = (v.T if stored_k_first else v).astype(f32)
        b = np.zeros((v.shape[0], qr.pitch(v.shape[1])), np.uint8)
        b[:, :v.shape[1]] = qr.encode(v)
        return QTensor.from_numpy(b, np.ones(qr.scale_shape(form, *v.shape), f32), v.shape[1], form)

    for fa, fb in forms(ta, tb):
        c = linalg.gemm_q_into(Tensor.empty(m, n), q(ai, ta, fa), q(bi, not tb, fb), trans_a=bool(ta), trans_b=bool(tb))
        assert np.array_equal(c.numpy(), (ai @ bi.T).astype(f32)), (fa, fb)


@pytest.mark.parametrize("m,n,k", [(1, 1000, 700), (24, 260, 256), (200, 131, 300)])
@pytest.mark.parametrize("act", ["identity", "relu", "sigmoid", "tanh"])
def test_bias_and_activation(m, n, k, act):
    a, av = operand(3, m, k, False, "rows")
    b, bv = operand(4, n, k, True, "tiles")
    av, bv = av / 64, bv / 64
    a, b = scaled(a, 1 / 64), scaled(b, 1 / 64)
    bias = np.random.default_rng(5).standard_normal(n).astype(f32)
    c = linalg.gemm_q_into(Tensor.empty(m, n), a, b, bias=Tensor(bias), act=act).numpy().astype(np.float64)
    z = av @ bv.T + bias.astype(np.float64)
    want = {"identity": lambda: z, "relu": lambda: np.maximum(z, 0), "sigmoid": lambda: 1 / (1 + np.exp(-z)),
            "tanh": lambda: np.tanh(z)}[act]()
    assert np.all(np.abs(c - want) <= bound(av, bv) + 2.0 ** -24 * np.abs(z) + 4e-7 * np.abs(want) + 1e-30)


def scaled(t: QTensor, factor: float) -> QTensor:
    return QTensor.from_numpy(t.numpy(), t.scales.numpy() * f32(factor), t.dims[1], t.blocks)


@pytest.mark.parametrize("m,n,k", [(70, 190, 500), (3, 700, 900), (1540, 1700, 260)])
def test_scales_may_be_any_values(m, n, k):
    rng = np.random.default_rng(9)
    a, _ = operand(6, m, k, False, "rows")
    b, _ = operand(7, n, k, False, "rows")
    sa, sb = rng.uniform(0.1, 3, a.scale_dims).astype(f32), rng.uniform(-2, 2, b.scale_dims).astype(f32)
    qa, qb = a.numpy(), b.numpy()
    av, bv = qr.values(qa, sa, "rows", k), qr.values(qb, sb, "rows", k)
    ta, tb = QTensor.from_numpy(qa, sa, k, "rows"), QTensor.from_numpy(qb, sb, k, "rows")
    assert ta.any_scales and tb.any_scales and not a.any_scales
    c = linalg.gemm_q_into(Tensor.empty(m, n), ta, tb, trans_b=True).numpy()
    assert np.all(np.abs(c - av @ bv.T) <= bound(av, bv))
    # one operand of each kind
    c = linalg.gemm_q_into(Tensor.empty(m, n), a, tb, trans_b=True).numpy()
    av = qr.values(qa, a.scales.numpy(), "rows", k)
    assert np.all(np.abs(c - av @ bv.T) <= bound(av, bv))
    # and read back
    assert np.array_equal(linalg.dequantize(tb).numpy(), (qr.TABLE[qb[:, :k]].astype(f32) * qr.spread(sb, "rows", n, k)))


@pytest.mark.parametrize("m,n,k", [(65, 130, 1500), (1540, 1700, 700)])
def test_scales_far_apart(m, n, k):
    # scales from one end of the range of powers of two to the other, in one sum and in one product
    rng = np.random.default_rng(19)
    a, _ = operand(6, m, k, False, "rows")
    b, _ = operand(7, n, k, False, "rows")
    sa = (2.0 ** rng.integers(-100, 60, a.scale_dims)).astype(f32)
    sb = (2.0 ** rng.integers(-20, 40, b.scale_dims)).astype(f32)
    ta, tb = QTensor.from_numpy(a.numpy(), sa, k, "rows"), QTensor.from_numpy(b.numpy(), sb, k, "rows")
    assert not ta.any_scales and not tb.any_scales
    av, bv = qr.values(a.numpy(), sa, "rows", k), qr.values(b.numpy(), sb, "rows", k)
    c = linalg.gemm_q_into(Tensor.empty(m, n), ta, tb, trans_b=True).numpy()
    assert np.all(np.abs(c - av @ bv.T) <= bound(av, bv) + 1e-37)


def test_nan_reaches_its_row_and_no_other():
    m, n, k = 130, 140, 300
    a, av = operand(8, m, k, False, "rows")
    b, bv = operand(9, n, k, True, "tiles")
    q = a.numpy()
    q[17, 299] = 0x7F
    c = linalg.gemm_q_into(Tensor.empty(m, n), QTensor.from_numpy(q, a.scales.numpy(), k, "rows"), b).numpy()
    assert np.all(np.isnan(c[17]))
    rest = np.arange(m) != 17
    assert np.all(np.abs(c[rest] - (av @ bv.T)[rest]) <= bound(av, bv)[rest])


@pytest.mark.parametrize("m,n,k", [(5, 400, 1000), (300, 500, 700)])
def test_same_bits_every_time_and_nothing_written_outside(m, n, k):
    a, _ = operand(10, m, k, False, "rows")
    b, _ = operand(11, n, k, True, "tiles")
    # c between two guard bands, and not 16-byte aligned
    base = Tensor(np.full(m * n + 65, 7, f32))
    c = Tensor.from_device_ptr(base.data_ptr + 4 * 33, m, n)
    first = linalg.gemm_q_into(c, a, b).numpy().copy()
    for _ in range(3):
        assert np.array_equal(linalg.gemm_q_into(c, a, b).numpy(), first)
    assert np.array_equal(linalg.gemm_q_into(Tensor.empty(m, n), a, b).numpy(), first)
    whole = base.numpy()
    assert np.all(whole[:33] == 7) and np.all(whole[33 + m * n:] == 7)


def test_captured_product_replays_on_new_operands():
    m, n, k = 9, 300, 640
    a, av = operand(12, m, k, False, "rows")
    a2, av2 = operand(13, m, k, False, "rows")
    b, bv = operand(14, n, k, True, "tiles")
    x, c = Tensor.empty(m, k), Tensor.empty(m, n)

    def step():
        linalg.gemm_q_into(c, linalg.quantize(x, "rows"), b)

    linalg.dequantize(a, x)
    g = cb.StepGraph(step)
    for t, v in ((a2, av2), (a, av)):
        linalg.dequantize(t, x)       # quantizing these values again gives the same bytes
        g.replay()
        cb.sync()
        assert np.all(np.abs(c.numpy() - v @ bv.T) <= bound(v, bv))
    g.close()


def test_two_threads_at_once():
    from concurrent.futures import ThreadPoolExecutor
    m, n, k = 64, 512, 768
    a, av = operand(15, m, k, False, "rows")
    b, bv = operand(16, n, k, True, "tiles")
    out = [Tensor.empty(m, n) for _ in range(8)]
    with ThreadPoolExecutor(4) as pool:
        list(pool.map(lambda c: linalg.gemm_q_into(c, a, b), out))
    for c in out:
        assert np.all(np.abs(c.numpy() - av @ bv.T) <= bound(av, bv))


def test_library_refuses_what_does_not_fit():
    L = cb.lib()
    a, _ = operand(20, 64, 96, False, "rows")
    b, _ = operand(21, 32, 96, True, "tiles")
    c = Tensor.empty(64, 32)
    A, B = (a._h, a.scales._h), (b._h, b.scales._h)

    def call(code, c=c._h, A=A, fa=1, B=B, fb=3, m=64, n=32, k=96, ta=0, tb=0, bias=None, act=0):
        assert L.cleave_cuda_gemm_e4m3(c, *A, fa, *B, fb, m, n, k, ta, tb, bias, act) == -code
        assert L.cleave_cuda_last_error() == code
        L.cleave_cuda_clear_error()

    call(4, m=0)
    call(3, k=95)
    call(3, n=48)
    short, row = Tensor.empty(64, 31), Tensor.empty(31)
    call(3, c=short._h)
    call(3, fa=2)                                           # scales of another form
    call(4, fa=0)
    call(4, act=4)
    call(3, bias=row._h)
    call(2, bias=ctypes.c_void_p(0x1230))
    call(4, A=(c._h, a.scales._h))                          # f32 where bytes belong
    call(4, c=a._h)                                         # bytes where f32 belongs
    wide = Tensor.empty(64, 64)
    over = linalg.QTensor.from_device_ptr(wide.data_ptr, a.scales.data_ptr, 64, 96, "rows")
    c_over = Tensor.from_device_ptr(wide.data_ptr + 64, 64, 32)
    call(4, c=c_over._h, A=(over._h, over.scales._h))       # the output over an operand
    cols, _ = operand(22, 64, 96, False, "cols")
    call(4, A=(cols._h, cols.scales._h), fa=2)              # blocks across the contraction
    rows, _ = operand(23, 32, 96, True, "rows")
    call(4, B=(rows._h, rows.scales._h), fb=1)
    assert L.cleave_cuda_gemm_e4m3(c._h, *A, 1, *B, 3, 64, 32, 96, 0, 0, None, 0) == 0
    with pytest.raises(TypeError):
        linalg.gemm_q_into(c, a, b, trans_b=True)
    with pytest.raises(TypeError):
        linalg.gemm_q_into(c, cols, b)
    cb.sync()
