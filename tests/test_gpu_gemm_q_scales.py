"""Scales at both ends of their range: wherever the result of an 8-bit product fits f32, the scales' own product, or one scale's with
a block's sum, may not leave the range on the way.

Bound: that of test_gpu_gemm_q.py.  Below 2^-126 a rounding is absolute, at most 2^-150: two a k-block (the scaled sum, the running
sum) and one a rank of a split.  Where the tensor pipe applies the scales its truncating adds lose up to 2^-149 each there; as in that
bound, every term of a sum counts as an add of its own: k * 2^-149."""
import numpy as np
import pytest

import _quant_ref as qr
from cleave_b200 import linalg
from cleave_b200.linalg import QTensor, Tensor
from test_gpu_gemm_q import bound, forms

pytestmark = pytest.mark.gpu
f32 = np.float32
# (exponents of A's scales, of B's, what the bytes are); "small": sums of a few 2^-18; "apart": every product is 0
CASES = [((70, 70), (60, 60), "small"), ((127, 127), (8, 10), "small"), ((8, 10), (127, 127), "small"), ((64, 64), (64, 64), "apart"),
         ((127, 127), (127, 127), "apart"), ((108, 110), (-20, -18), "full"), ((-20, -18), (108, 110), "full"),
         ((-126, -120), (60, 80), "full"), ((60, 80), (-126, -120), "full"), ((-100, -100), (-52, -50), "full"),
         ((-126, -126), (-28, -26), "full"), ((-126, 70), (-70, 126), "full")]
# no split and a split, rows of C and of its transpose on the MMA's 128 rows, 16 to 128 columns
ONE_CTA = [(100, 130, 300), (7, 300, 300), (30, 300, 1500), (300, 60, 260)]


def operand(rng, free, k, stored_k_first, form, exponents, kind, side):
    shape = (k, free) if stored_k_first else (free, k)
    if kind == "full":
        q = rng.integers(0, 256, (shape[0], qr.pitch(shape[1])), dtype=np.uint8)
        q[(q & 0x7F) == 0x7F] = 0
    else:
        q = np.where(rng.random((shape[0], qr.pitch(shape[1]))) < 0.25, rng.choice([0x01, 0x81], (shape[0], qr.pitch(shape[1]))), 0)
        if kind == "apart":   # A has its bytes at even places of the contraction, B at odd ones
            at = np.arange(side, k, 2)
            q[at if stored_k_first else slice(None), slice(None) if stored_k_first else at] = 0
        q = q.astype(np.uint8)
    s = 2.0 ** rng.integers(exponents[0], exponents[1] + 1, qr.scale_shape(form, *shape)).astype(np.float64)
    v = qr.values(q, s, form, shape[1])
    t = QTensor.from_numpy(q, s.astype(f32), shape[1], form)
    assert not t.any_scales
    return t, (v.T if stored_k_first else v)


def check(m, n, k, ta, tb, fa, fb, case, any_scales=False, pairs=False):
    rng = np.random.default_rng(m + n)
    ea, eb, kind = case
    a, av = operand(rng, m, k, ta, fa, ea, kind, 0)
    b, bv = operand(rng, n, k, not tb, fb, eb, kind, 1)
    if any_scales:
        for t in (a, b):
            t.any_scales, t.form = True, t.form | linalg.SCALES_ANY
    c = linalg.gemm_q_into(Tensor.filled(np.nan, m, n), a, b, trans_a=bool(ta), trans_b=bool(tb)).numpy().astype(np.float64)
    fits = np.abs(av) @ np.abs(bv).T <= 2.0 ** 126     # no partial sum can overflow
    assert fits.all() or ea == CASES[-1][0]
    err, most = np.abs(c - av @ bv.T), bound(av, bv) + (2 * -(-k // 128) + 8) * 2.0 ** -150 + (k * 2.0 ** -149 if pairs else 0.0)
    worse = fits & ~(err <= most)
    assert not worse.any(), (fa, fb, int(worse.sum()), c[worse][:4], (av @ bv.T)[worse][:4])


@pytest.mark.parametrize("m,n,k", ONE_CTA)
@pytest.mark.parametrize("ta,tb", [(0, 0), (1, 1)])
@pytest.mark.parametrize("case", CASES)
def test_scales_at_both_ends(m, n, k, ta, tb, case):
    for fa, fb in forms(ta, tb):
        check(m, n, k, ta, tb, fa, fb, case)


@pytest.mark.parametrize("any_scales", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_scales_at_both_ends_large(case, any_scales):
    # enough tiles for the kernel on CTA pairs, unless the tensors are marked
    for fa, fb in forms(0, 0):
        check(1540, 1300, 260, 0, 0, fa, fb, case, any_scales, pairs=not any_scales)


@pytest.mark.parametrize("m,n", [(70, 190), (9, 190)])
def test_marked_scales_beyond_the_powers_of_two(m, n):
    # marked tensors may hold any f32 scales: subnormal ones, negative ones, zero
    k, rng = 700, np.random.default_rng(3)
    a, _ = operand(rng, m, k, False, "rows", (0, 0), "full", 0)
    b, _ = operand(rng, n, k, False, "rows", (0, 0), "full", 1)
    sa = rng.choice([2.0 ** -149, 3.0 * 2.0 ** -140, -1.25 * 2.0 ** -126, 0.0, 1.5 * 2.0 ** -101, -1.5 * 2.0 ** -99], a.scale_dims).astype(f32)
    sb = (rng.uniform(1, 2, b.scale_dims) * 2.0 ** rng.integers(90, 100, b.scale_dims)).astype(f32)
    for x, y in ((sa, sb), (np.abs(sb).reshape(-1)[np.arange(sa.size) % sb.size].reshape(sa.shape),
                            sa.reshape(-1)[np.arange(sb.size) % sa.size].reshape(sb.shape))):
        ta, tb = QTensor.from_numpy(a.numpy(), x, k, "rows"), QTensor.from_numpy(b.numpy(), y, k, "rows")
        av, bv = qr.values(a.numpy(), x, "rows", k), qr.values(b.numpy(), y, "rows", k)
        c = linalg.gemm_q_into(Tensor.filled(np.nan, m, n), ta, tb, trans_b=True).numpy().astype(np.float64)
        assert np.all(np.abs(c - av @ bv.T) <= bound(av, bv) + (2 * -(-k // 128) + 8) * 2.0 ** -150)
