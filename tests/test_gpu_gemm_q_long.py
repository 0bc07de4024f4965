"""The 8-bit product where its pipelines go round: long contractions, several tiles for a cluster, more k-blocks than a ring holds.

Bytes and scales are drawn at random, a scale for every block, so that one taken from another block shows.  The bound is that of
test_gpu_gemm_q.py."""
import numpy as np
import pytest

import _quant_ref as qr
from cleave_b200 import linalg
from cleave_b200.linalg import QTensor, Tensor
from test_gpu_gemm_q import TRANS, bound, forms

pytestmark = pytest.mark.gpu
f32 = np.float32


def operand(seed, free, k, stored_k_first, form, centre=0, any_scales=False):
    rng = np.random.default_rng(seed)
    shape = (k, free) if stored_k_first else (free, k)
    q = rng.integers(0, 256, (shape[0], qr.pitch(shape[1])), dtype=np.uint8)
    q[:, :shape[1]][(q[:, :shape[1]] & 0x7F) == 0x7F] = 0
    s = (2.0 ** (centre + rng.integers(-3, 4, qr.scale_shape(form, *shape)))).astype(f32)
    if any_scales:
        s *= rng.uniform(0.5, 2, s.shape).astype(f32)
    t = QTensor.from_numpy(q, s, shape[1], form)
    assert t.any_scales == any_scales

    def rows(at):
        """Values of those of the free extent, [len(at), k]."""
        every = qr.spread(s, form, *shape)
        return (qr.TABLE[q[:, at]] * every[:, at]).T if stored_k_first else qr.TABLE[q[at, :k]] * every[at]
    return t, rows


def check(m, n, k, ta, tb, fa, fb, act="identity", bias=False, any_scales=False):
    a, a_rows = operand(1, m, k, ta, fa, -9 if act != "identity" else 0, any_scales)
    b, b_rows = operand(2, n, k, not tb, fb, -9 if act != "identity" else 0, any_scales)
    bv = np.random.default_rng(5).standard_normal(n).astype(f32) if bias else None
    c = linalg.gemm_q_into(Tensor.filled(np.nan, m, n), a, b, trans_a=bool(ta), trans_b=bool(tb),
                           bias=Tensor(bv) if bias else None, act=act).numpy()
    assert not np.isnan(c).any()
    rows = np.unique(np.concatenate([np.arange(0, m, max(1, m // 150)), [m - 1]]))   # of every tile
    av, bw = a_rows(rows), b_rows(np.arange(n))
    z = av @ bw.T + (bv.astype(np.float64) if bias else 0.0)
    want = {"identity": lambda: z, "sigmoid": lambda: 1 / (1 + np.exp(-z)), "tanh": lambda: np.tanh(z), "relu": lambda: np.maximum(z, 0)}[act]()
    most = bound(av, bw) + 2.0 ** -24 * np.abs(z) + (4e-7 * np.abs(want) if act in ("sigmoid", "tanh") else 0.0)
    err = np.abs(c[rows].astype(np.float64) - want)
    assert np.all(err <= most), (fa, fb, float(np.max(err / most)))


# CTA pairs: k-blocks that are no multiple of 4 (scale words) or 8 (a chunk of the accumulator), one to three tiles a cluster
@pytest.mark.parametrize("m,n,k", [(1300, 1281, 1100), (1281, 1026, 2200), (1300, 1281, 4200), (2320, 2500, 600), (2310, 4100, 1100)])
@pytest.mark.parametrize("ta,tb", TRANS)
def test_pairs_over_long_contractions_and_several_tiles(m, n, k, ta, tb):
    for fa, fb in forms(ta, tb):
        check(m, n, k, ta, tb, fa, fb)


@pytest.mark.parametrize("m,n,k", [(1300, 1281, 1100), (2310, 4100, 600)])
@pytest.mark.parametrize("act", ["tanh", "sigmoid"])
def test_pairs_with_bias_and_activation(m, n, k, act):
    check(m, n, k, 0, 0, "rows", "tiles", act, True)
    check(m, n, k, 1, 1, "tiles", "rows", act, True)


# one CTA a tile: 110 k-blocks over eight CTAs, 13 and 14 each, on rings of 3 to 5 stages and 6 to 8 scale slots
@pytest.mark.parametrize("m,n,k", [(5, 200, 14000), (30, 200, 14000), (60, 200, 14000), (200, 130, 14000)])
@pytest.mark.parametrize("ta,tb", TRANS)
def test_one_cta_kernel_over_many_blocks(m, n, k, ta, tb):
    for fa, fb in forms(ta, tb):
        check(m, n, k, ta, tb, fa, fb, bias=True)


@pytest.mark.parametrize("m,n,k", [(100, 20000, 1700), (20, 19200, 1700)])
def test_one_cta_kernel_without_a_split(m, n, k):
    check(m, n, k, 0, 0, "rows", "tiles", "tanh", True)
    check(m, n, k, 0, 1, "tiles", "rows")


@pytest.mark.parametrize("m,n,k", [(1300, 1281, 1700), (40, 900, 9000)])
@pytest.mark.parametrize("ta,tb", TRANS)
def test_any_scales_over_many_blocks(m, n, k, ta, tb):
    for fa, fb in forms(ta, tb):
        check(m, n, k, ta, tb, fa, fb, any_scales=True)
