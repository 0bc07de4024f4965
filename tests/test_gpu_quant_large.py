"""8-bit tensors at the far ends of the sizes: more than 2^31 elements, sides of 2^31 - 1, more column blocks than the column sums
have counters, many row blocks.  Only slices are compared, against the numpy yardstick."""
import numpy as np
import pytest
import torch

import _quant_ref as qr
import cleave_b200 as cb
from cleave_b200 import linalg, nn
from cleave_b200.linalg import QTensor, Tensor
from test_gpu_quant import FORMS, SIZES, assert_colsum, checkpoint, wide

pytestmark = pytest.mark.gpu
f32 = np.float32


def tensor(t: torch.Tensor) -> Tensor:
    v = Tensor.from_device_ptr(t.data_ptr(), *t.shape)
    v._owner = t
    return v


@pytest.fixture(autouse=True)
def give_memory_back():
    yield
    torch.cuda.empty_cache()


class Quantized:
    """An 8-bit tensor over torch memory, of which slices can be looked at."""

    def __init__(self, rows, cols, form):
        self.bytes = torch.empty(rows, qr.pitch(cols), dtype=torch.uint8, device="cuda")
        self.scales = torch.empty(qr.scale_shape(form, rows, cols), dtype=torch.float32, device="cuda")
        self.q = QTensor.from_device_ptr(self.bytes.data_ptr(), self.scales.data_ptr(), rows, cols, form)
        self.form, self.rows, self.cols = form, rows, cols

    def part(self, r0, r1, c0, c1):
        """Bytes and scales of a slice that starts at a block's corner."""
        b = self.bytes[r0:r1, c0:c1].cpu().numpy()
        rb, cb_ = slice(r0 // 128, -(-r1 // 128)), slice(c0 // 128, -(-c1 // 128))
        s = {"rows": (cb_, slice(r0, r1)), "cols": (rb, slice(c0, c1)), "tiles": (rb, cb_)}[self.form]
        return b, self.scales[s].cpu().numpy()


def check_slice(t: Quantized, values: np.ndarray, r0, r1, c0, c1):
    b, s = t.part(r0, r1, c0, c1)
    q, want_s = qr.quantize(values, t.form)
    assert np.array_equal(s, want_s)
    assert np.array_equal(b, q[:, :c1 - c0])


def settled():
    torch.cuda.synchronize()
    cb.sync()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_f32_gradient_and_column_sums_together(rows, cols, form):
    y, y_val = checkpoint(rows, cols, "sigmoid", form)
    g = wide(rows, cols, 11)
    dz, db = Tensor.empty(rows, cols), Tensor.empty(cols)
    nn.act_bwd_q(y, Tensor(g), "sigmoid", dz=dz, db=db)
    want = qr.act_bwd_f32(y_val, g, "sigmoid")
    assert np.array_equal(dz.numpy(), want)
    assert_colsum(db.numpy(), want)


@pytest.mark.parametrize("rows,cols", [(129, 128 * 4096 + 130), (128 * 700 + 5, 131)])
@pytest.mark.parametrize("quantized", [False, True])
def test_column_sums_of_many_blocks(rows, cols, quantized):
    gen = torch.Generator(device="cuda").manual_seed(rows)
    y = Quantized(rows, cols, "tiles")
    y.bytes.copy_(torch.randint(0, 0x40, y.bytes.shape, generator=gen, device="cuda", dtype=torch.uint8))   # 0 .. 2
    y.scales.fill_(1.0)
    g = torch.randn(rows, cols, generator=gen, device="cuda")
    out = Quantized(rows, cols, "cols")
    db = torch.empty(cols, device="cuda")
    settled()
    nn.act_bwd_q(y.q, tensor(g), "relu", *([out.q] if quantized else []), db=tensor(db))
    settled()
    dz = torch.where(y.bytes[:, :cols] > 0, g, torch.zeros_like(g))
    assert_colsum(db.cpu().numpy(), dz.cpu().numpy())


def test_more_elements_than_32_bits_count():
    rows, cols = 66001, 32771            # 2.16e9
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    forms = [Quantized(rows, cols, f) for f in FORMS]
    dz = torch.full((rows, cols), float("nan"), device="cuda")
    db = torch.empty(cols, device="cuda")
    settled()
    linalg.quantize_into(tensor(x), *[t.q for t in forms])
    settled()
    r0, c0 = rows // 128 * 128, cols // 128 * 128
    corners = [(r0, rows, c0, cols), (r0, rows, 0, 256), (r0 - 128, r0, c0 - 256, cols), (0, 128, c0, cols)]
    for t in forms:
        for c in corners:
            check_slice(t, x[c[0]:c[1], c[2]:c[3]].cpu().numpy(), *c)
        linalg.dequantize(t.q, tensor(dz))
        settled()
        for r0_, r1, c0_, c1 in corners:
            b, s = t.part(r0_, r1, c0_, c1)
            assert np.array_equal(dz[r0_:r1, c0_:c1].cpu().numpy(), qr.values(b, s, t.form, c1 - c0_))
        nn.act_bwd_q(t.q, tensor(x), "tanh", dz=tensor(dz), db=tensor(db))
        settled()
        for r0_, r1, c0_, c1 in corners:
            b, s = t.part(r0_, r1, c0_, c1)
            want = qr.act_bwd_f32(qr.values(b, s, t.form, c1 - c0_).astype(f32), x[r0_:r1, c0_:c1].cpu().numpy(), "tanh")
            assert np.array_equal(dz[r0_:r1, c0_:c1].cpu().numpy(), want)
        for lo in (0, cols - 300):
            assert_colsum(db[lo:lo + 300].cpu().numpy(), dz[:, lo:lo + 300].cpu().numpy())


def test_product_with_more_elements_than_32_bits_count():
    rows, cols, k = 66001, 32771, 40
    gen = torch.Generator(device="cuda").manual_seed(2)
    a = torch.randint(-3, 4, (rows, k), generator=gen, device="cuda").float()     # small integers: every form of the product is exact
    b = torch.randint(-3, 4, (k, cols), generator=gen, device="cuda").float()
    c = torch.full((rows, cols), float("nan"), device="cuda")
    settled()
    linalg.gemm_q_into(tensor(c), linalg.quantize(tensor(a), "rows"), linalg.quantize(tensor(b), "cols"))
    settled()
    for r in (slice(0, 128), slice(rows // 2, rows // 2 + 128), slice(rows - 150, rows)):
        assert np.array_equal(c[r].cpu().numpy(), a[r].cpu().numpy() @ b.cpu().numpy())


LONGEST = 2 ** 31 - 1


@pytest.mark.parametrize("shape", [(1, LONGEST), (LONGEST, 1)])
def test_longest_sides(shape):
    rows, cols = shape
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(shape, generator=gen, device="cuda")
    t = Quantized(rows, cols, "tiles")
    back = torch.full(shape, float("nan"), device="cuda")
    settled()
    linalg.quantize_into(tensor(x), t.q)
    linalg.dequantize(t.q, tensor(back))
    settled()
    ends = [(0, 256), (LONGEST // 128 * 128 - 256, LONGEST)]
    cuts = [(0, 1, *e) if rows == 1 else (*e, 0, 1) for e in ends]
    for r0, r1, c0, c1 in cuts:
        check_slice(t, x[r0:r1, c0:c1].cpu().numpy(), r0, r1, c0, c1)
        b, s = t.part(r0, r1, c0, c1)
        assert np.array_equal(back[r0:r1, c0:c1].cpu().numpy(), qr.values(b, s, "tiles", c1 - c0))
    nn.act_bwd_q(t.q, tensor(x), "identity", dz=tensor(back))
    settled()
    for r0, r1, c0, c1 in cuts:
        assert np.array_equal(back[r0:r1, c0:c1].cpu().numpy(), x[r0:r1, c0:c1].cpu().numpy())
