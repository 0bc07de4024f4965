"""The block-scaled 8-bit form in plain numpy, values in 64 bits: the yardstick of the 8-bit operator tests.

e4m3: sign, 4 exponent bits (bias 7), 3 mantissa bits; exponent 0 is subnormal (steps of 2^-9), 0x7F / 0xFF are NaN, the
largest value is 448 and there is no infinity.
"""
import numpy as np

BLOCK = 128


def decode_table() -> np.ndarray:
    t = np.empty(256, np.float64)
    for b in range(256):
        sign, e, m = (-1.0 if b & 0x80 else 1.0), (b >> 3) & 15, b & 7
        if e == 15 and m == 7:
            t[b] = np.nan
        else:
            t[b] = sign * (m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    return t


TABLE = decode_table()


def encode(v: np.ndarray) -> np.ndarray:
    """e4m3 bytes of values of magnitude at most 448, round half to even; non-finite values become NaN."""
    v = np.asarray(v, np.float64)
    fine = np.isfinite(v)
    a = np.abs(np.where(fine, v, 0.0))
    assert a.size == 0 or a.max() <= 448.0
    e = np.clip(np.floor(np.log2(np.maximum(a, 2.0 ** -20))), -6, 8).astype(np.int64)
    n = np.rint(a / 2.0 ** (e - 3).astype(np.float64)).astype(np.int64)     # 8 .. 16 in the normal range, 0 .. 8 below it
    up = n == 16
    e, n = np.where(up, e + 1, e), np.where(up, 8, n)
    b = np.where(n < 8, n, ((e + 7) << 3) | (n - 8))
    b = np.where(fine, b, 0x7F)
    return (b | (np.signbit(v).astype(np.int64) << 7)).astype(np.uint8)


def pitch(cols: int) -> int:
    return -(-cols // 16) * 16


def _block(form):
    return {"rows": (1, BLOCK), "cols": (BLOCK, 1), "tiles": (BLOCK, BLOCK)}[form]


def scale_shape(form, rows, cols):
    rb, cb = -(-rows // BLOCK), -(-cols // BLOCK)
    return {"rows": (cb, rows), "cols": (rb, cols), "tiles": (rb, cb)}[form]


def spread(s: np.ndarray, form: str, rows: int, cols: int) -> np.ndarray:
    """Each element's scale."""
    s = s.T if form == "rows" else s
    h, w = _block(form)
    return s[np.arange(rows)[:, None] // h, np.arange(cols)[None, :] // w]


def quantize(x: np.ndarray, form: str):
    """(bytes [rows, pitch], scales f32): scale = 2^e, the smallest with amax <= 448 * 2^e, e in [-126, 120]."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    h, w = _block(form)
    rb, cb = -(-rows // h), -(-cols // w)
    a = np.zeros((rb * h, cb * w))
    a[:rows, :cols] = np.where(np.isfinite(x), np.abs(x), 0.0)
    amax = a.reshape(rb, h, cb, w).max(axis=(1, 3))
    e = np.full(amax.shape, -126)
    for cand in range(120, -127, -1):
        e = np.where(amax <= 448.0 * 2.0 ** cand, cand, e)
    s = 2.0 ** e.astype(np.float64)
    s = s.T if form == "rows" else s
    q = np.zeros((rows, pitch(cols)), np.uint8)
    q[:, :cols] = encode(x / spread(s, form, rows, cols))
    return q, np.ascontiguousarray(s).astype(np.float32)


def values(q: np.ndarray, s: np.ndarray, form: str, cols: int) -> np.ndarray:
    return TABLE[q[:, :cols]] * spread(np.asarray(s, np.float64), form, q.shape[0], cols)


# dz = act'(y) * g, each f32 operation rounded as the library's derivative forms round it
def act_bwd_f32(y: np.ndarray, g: np.ndarray, act: str) -> np.ndarray:
    y, g, one = np.asarray(y, np.float32), np.asarray(g, np.float32), np.float32(1)
    if act == "tanh":
        return (one - y * y) * g
    if act == "sigmoid":
        return (y * (one - y)) * g
    if act == "relu":
        return np.where(y > 0, g, np.float32(0))
    return g.copy()
