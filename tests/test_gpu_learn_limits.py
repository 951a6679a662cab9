"""The learning operators at more rows and columns than a launch's 2^32 threads hold at a
workgroup or a wave each."""

import numpy as np
import pytest

from tests import learn_ref as R

pytestmark = pytest.mark.gpu
U = R.U32
NONE = 0xFFFFFFFF


@pytest.fixture(scope="module")
def dev():
    from emeans_amd import HipDevice
    d = HipDevice()
    yield d
    d.close()


def test_norm_of_very_many_short_rows(dev):
    """Rows shorter than a vector: a workgroup each, in both passes. Sums over the rows are
    64 chains in f32."""
    from emeans_amd import F32
    rows, d = (1 << 24) + 3, 2
    r = np.random.default_rng(1)
    x = r.standard_normal((rows, d), dtype=np.float32)
    dy = r.standard_normal((rows, d), dtype=np.float32)
    w, b = np.array([1.5, -0.5], np.float32), np.array([0.25, 2.0], np.float32)
    xb, wb, bb, y = dev.upload_f32(x), dev.upload_f32(w), dev.upload_f32(b), dev.zeros(rows * d, F32)
    mean, rstd = dev.zeros(rows, F32), dev.zeros(rows, F32)
    dev.layer_norm(xb, rows, d, wb, bb, y, mean, rstd)
    want, m64, s64, h = R.layer_norm(x.astype(float), w.astype(float), b.astype(float), 1e-5)
    # A difference of two elements and its root: a dozen roundings; the mean's error moves
    # both differences by a rounding of the larger element.
    tol = 32 * U * (1 + np.abs(want)) + 4 * U * (np.abs(x).max(1) * s64)[:, None]
    assert np.all(np.abs(dev.read(y).reshape(rows, d) - want) <= 2 * tol)
    assert np.all(np.abs(dev.read(mean) - m64) <= 4 * U * np.abs(x).max(1))
    dx, dw, db = dev.zeros(rows * d, F32), dev.zeros(d, F32), dev.zeros(d, F32)
    dev.layer_norm_grad(dev.upload_f32(dy), xb, rows, d, wb, mean, rstd, dx, dw, db)
    want, dw64, db64 = R.layer_norm_grad(dy.astype(float), h, s64, w.astype(float))
    dh = 32 * U * 2 + 4 * U * (np.abs(x).max(1) * s64)
    off = s64 * 2 * np.abs(dy).max(1) * 1.5 * (32 * U + 8 * dh)
    assert np.all(np.abs(dev.read(dx).reshape(rows, d) - want) <= off[:, None])
    chain = (rows / 64 + 64) * U
    ady = np.abs(dy.astype(float))
    assert np.all(np.abs(dev.read(dw) - dw64) <= chain * ady.sum(0) * 2 + (ady * dh[:, None]).sum(0))
    assert np.all(np.abs(dev.read(db) - db64) <= chain * ady.sum(0))


def test_norm_gradient_of_very_many_columns(dev):
    from emeans_amd import F32
    d = (1 << 25) + 5
    r = np.random.default_rng(2)
    x = r.standard_normal(d, dtype=np.float32)
    dy = r.standard_normal(d, dtype=np.float32)
    xb, dyb = dev.upload_f32(x), dev.upload_f32(dy)
    mean, rstd = dev.upload_f32([x.mean(dtype=float)]), dev.upload_f32([1.0 / x.std(dtype=float)])
    dw, db = dev.zeros(d, F32), dev.zeros(d, F32)
    dev.layer_norm_grad(dyb, xb, 1, d, None, mean, rstd, None, dw, db)
    m, s = float(dev.read(mean)[0]), float(dev.read(rstd)[0])
    want = dy * ((x.astype(float) - m) * s)
    assert np.all(np.abs(dev.read(dw) - want) <= 4 * U * np.abs(dy) * s * (np.abs(x) + abs(m)))
    assert np.array_equal(dev.read(db), dy)


def test_cross_entropy_of_very_many_rows(dev):
    """Rows that are laid out for the tiles, a wave each."""
    from emeans_amd import F16, F32
    n, k = (1 << 26) + 5, 2
    r = np.random.default_rng(3)
    x = r.standard_normal(n, dtype=np.float32).astype(np.float16)
    lab = r.integers(0, k, n, dtype=np.uint32)
    lab[::1001] = NONE
    w = np.array([1.5, -0.5], np.float16)
    xb, wb, lb = dev.zeros(n, F16), dev.zeros(k, F16), dev.upload_u32(lab)
    dev.write(xb, 0, x)
    dev.write(wb, 0, w)
    loss, lse = dev.zeros(n, F32), dev.zeros(n, F32)
    dev.cross_entropy(xb, n, 1, wb, k, lb, loss, lse)
    got, got_lse = dev.read(loss), dev.read(lse)
    at = np.concatenate([np.arange(2000), np.arange(n - 2000, n), r.integers(0, n, 20_000)])
    want, lse64, _, z = R.cross_entropy(x[at, None].astype(float), w[:, None].astype(float), lab[at], 1.0)
    tol = 16 * U * (1 + np.abs(z).max(1))
    assert np.all(np.abs(got[at] - want) <= tol) and np.all(np.abs(got_lse[at] - lse64) <= tol)
    assert np.all(got_lse != 0.0) and not got[::1001].any()


def test_zeros_of_more_than_a_launch_of_words(dev):
    """On memory that was not zero before, where the allocator gives the same again."""
    from emeans_amd import F8
    n = (1 << 34) + 1027
    for _ in range(2):
        b = dev.zeros(n, F8)
        for lo in (0, (1 << 34) - 1500, n - 1027):
            assert not dev.read(b, (lo, lo + 1000)).any()
            dev.write(b, lo, np.full(1000, 7, np.uint8))
        del b
