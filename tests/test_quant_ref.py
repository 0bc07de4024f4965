"""The 8-bit yardstick itself, on the CPU: against torch's e4m3 conversions and by its own definition."""
import numpy as np
import pytest
import torch

import _quant_ref as qr


def test_decode_table_is_torchs_e4m3():
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(np.isnan(t), np.isnan(qr.TABLE)) and np.array_equal(t[~np.isnan(t)], qr.TABLE[~np.isnan(t)])


def test_encode_rounds_half_to_even_and_round_trips():
    fine = ~np.isnan(qr.TABLE)
    assert np.array_equal(qr.encode(qr.TABLE[fine]), np.arange(256, dtype=np.uint8)[fine])
    rng = np.random.default_rng(1)
    v = np.concatenate([rng.uniform(-448, 448, 5000), rng.uniform(-0.05, 0.05, 5000),
                        rng.integers(0, 2 ** 13, 4000) * 2.0 ** -11, [2.0 ** -10, 1.5 * 2.0 ** -9, 432.0, 447.9]]).astype(np.float32)
    want = torch.from_numpy(v).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(qr.encode(v), want)
    assert list(qr.encode(np.array([np.nan, np.inf]))) == [0x7F, 0x7F] and qr.encode(np.array([-np.inf]))[0] == 0xFF


@pytest.mark.parametrize("form", ["rows", "cols", "tiles"])
def test_quantize_error_is_at_most_half_a_step(form):
    rng = np.random.default_rng(2)
    x = (rng.standard_normal((200, 300)) * 2.0 ** rng.integers(-20, 20, (200, 1))).astype(np.float32)
    q, s = qr.quantize(x, form)
    assert q.shape == (200, 304) and s.shape == qr.scale_shape(form, 200, 300)
    v, each = qr.values(q, s, form, 300), qr.spread(s, form, 200, 300)
    # half a step: 2^-4 of the value, or of the smallest normal 2^-6 (in units of the scale)
    assert np.all(np.abs(v - x) <= 2.0 ** -4 * np.maximum(np.abs(x), 2.0 ** -6 * each))
