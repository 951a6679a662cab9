"""Long sums of the RMS norm: rows of millions of elements, and millions of short rows, whose terms
are all alike (roundings of a sum of equal terms go the same way)."""

import numpy as np
import pytest

from tests import learn_ref as R

pytestmark = pytest.mark.gpu
EPS = 1e-6
U = R.U32


@pytest.fixture(scope="module")
def dev():
    from emeans_amd import HipDevice
    d = HipDevice()
    yield d
    d.close()


def _rstd(v):
    return 1 / np.sqrt(float(np.float32(v)) ** 2 + EPS)


@pytest.mark.parametrize("d", [9001, 1 << 20, 1 << 24])
def test_rows_of_equal_elements(dev, d):
    """A thread's sum is exact, or all but: 256 of them join in 8 roundings and 3 more, with the
    quotient, the root and the product within 16."""
    from emeans_amd import F32
    x = np.full((2, d), 1.1, np.float32)
    x[1] = -0.7
    b, y, rstd = dev.upload_f32(x), dev.zeros(2 * d, F32), dev.zeros(2, F32)
    dev.rms_norm(b, 2, d, None, y, rstd=rstd, eps=EPS)
    want = np.array([_rstd(1.1), _rstd(0.7)])
    assert np.all(np.abs(dev.read(rstd) - want) <= 16 * U * want)
    got = dev.read(y).reshape(2, d).astype(float)
    ref = x[:, :1].astype(float) * want[:, None]
    assert np.all(np.abs(got - ref) <= 18 * U * np.abs(ref))
    # The gradient of equal elements, g - u mean(g u), all but vanishes: what is left is roundings.
    dy, dx, dw = dev.upload_f32(np.full(2 * d, 0.9)), dev.zeros(2 * d, F32), dev.zeros(d, F32)
    dev.rms_norm_grad(dy, b, 2, d, None, rstd, dx, dw)
    g = np.abs(dev.read(dx).reshape(2, d)).max(1)
    assert np.all(g <= 0.9 * want * (EPS * want ** 2 + 64 * U))
    total = 0.9 * ref[:, 0].sum()
    assert np.all(np.abs(dev.read(dw) - total) <= 0.9 * 40 * U * np.abs(ref[:, 0]).sum())


@pytest.mark.parametrize("rows,d", [(1 << 22, 3), (5_000_001, 1)])
def test_many_short_rows(dev, rows, d):
    """dweight over millions of rows of fewer elements than a vector: the 64 shares' sums are added
    one by one."""
    from emeans_amd import F32
    x, dy = dev.upload_f32(np.full(rows * d, 1.1)), dev.upload_f32(np.full(rows * d, 0.9))
    y, rstd, dw = dev.zeros(rows * d, F32), dev.zeros(rows, F32), dev.zeros(d, F32)
    dev.rms_norm(x, rows, d, None, y, rstd=rstd, eps=EPS)
    dev.rms_norm_grad(dy, x, rows, d, None, rstd, None, dw)
    want = rows * float(np.float32(0.9)) * float(np.float32(1.1)) * _rstd(1.1)
    assert np.all(np.abs(dev.read(dw) - want) <= (64 + 24) * U * want)


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 1000, 9001])
def test_the_largest_sums_of_squares(dev, name, d):
    """Elements just below 2^64 / sqrt(d) have a norm; a row whose sum exceeds f32 has rstd 0."""
    from emeans_amd import F32
    r = np.random.default_rng(d)
    x = r.choice([-1.0, 1.0], (2, d)) * 0.98 * 2.0 ** 64 / np.sqrt(d)
    x[1] *= 1.1
    px, py = R.Padded(dev, x, name), R.Padded(dev, 0 * x, name)
    rstd = dev.zeros(2, F32)
    dev.rms_norm(px.buf, 2, d, None, py.buf, rstd=rstd, eps=EPS)
    v = px.value[0]
    want = 1 / np.sqrt((v * v).mean())
    got = dev.read(rstd)
    assert abs(got[0] - want) <= 2 * (d / 16 + 32) * U * want and got[1] == 0
    y = py.read()
    assert np.all(np.abs(y[0] - v * want) <= (2 * (d / 16 + 32) * U + R.UNIT[name]) * 1.01)
    assert not y[1].any()
