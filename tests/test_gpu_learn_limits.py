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


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_gradient_of_a_million_rows(dev, name):
    """The rows go in blocks, in the default workspace: rows and classes from their
    definition, dw over all rows."""
    from emeans_amd import F32
    n, d, k = 1_000_003, 24, 50
    r = np.random.default_rng(4)
    x = r.standard_normal((n, d), dtype=np.float32)
    w = r.standard_normal((k, d), dtype=np.float32) / np.sqrt(d)
    lab = r.integers(0, k, n, dtype=np.uint32)
    lab[::97] = NONE
    raw = R.encode(x, name)
    x64, w64 = R.decode(raw, name), R.decode(R.encode(w, name), name)
    kd = R.kind(name)
    xb, wb, lb = dev.zeros(n * d, kd), dev.zeros(k * d, kd), dev.upload_u32(lab)
    dev.write(xb, 0, raw.reshape(-1))
    dev.write(wb, 0, R.encode(w, name).reshape(-1))
    loss, lse = dev.zeros(n, F32), dev.zeros(n, F32)
    dx, dw = dev.zeros(n * d, kd), dev.zeros(k * d, kd)
    dev.cross_entropy(xb, n, d, wb, k, lb, loss, lse)
    # (Weights: a mean over a million rows is within bf16's and f16's range, but its
    # errors' bounds are easier to state without the common factor.)
    up = r.random(n, dtype=np.float32) + 0.5
    dev.cross_entropy_grad(xb, n, d, wb, k, lb, lse, dx, dw, gloss=dev.upload_f32(up))
    _, _, p, _ = R.cross_entropy(x64, w64, lab, 1.0)
    want_dx, want_dw, g = R.cross_entropy_grad(x64, w64, lab, 1.0, p, up.astype(float))
    # G: a unit of its type, and the softmax's own error, of a logit's sum of 24 terms.
    unit = {"f32": 2.0 ** -20, "bf16": 2.0 ** -8}[name]
    eg = 1.01 * unit * np.abs(g) + 2.0 ** -17 * p * up[:, None]
    eg[lab == NONE] = 0.0
    out = R.UNIT[name]
    tol = eg @ np.abs(w64) + 1.01 * out * np.abs(want_dx) + 1e-6
    assert np.all(np.abs(R.decode(dev.read(dx), name).reshape(n, d) - want_dx) <= tol)
    # Chains of f32 sums over a million rows; split by tiles, blocks and lanes.
    tol = eg.T @ np.abs(x64) + (n / 8 + 64) * U * (np.abs(g).T @ np.abs(x64)) / 16
    got = R.decode(dev.read(dw), name).reshape(k, d)
    assert np.all(np.abs(got - want_dw) <= tol + 1.01 * out * np.abs(want_dw))


def test_gradient_of_very_many_rows(dev):
    """Laid out, in blocks, at more rows than a launch holds waves; dw of two classes by the
    sums of its rows' own."""
    from emeans_amd import F16, F32
    n, k = (1 << 26) + 5, 2
    r = np.random.default_rng(6)
    x = r.standard_normal(n, dtype=np.float32).astype(np.float16)
    lab = r.integers(0, k, n, dtype=np.uint32)
    lab[::1001] = NONE
    w = np.array([1.5, -0.5], np.float16)
    xb, wb, lb = dev.zeros(n, F16), dev.zeros(k, F16), dev.upload_u32(lab)
    dev.write(xb, 0, x)
    dev.write(wb, 0, w)
    loss, lse, dx, dw = dev.zeros(n, F32), dev.zeros(n, F32), dev.zeros(n, F16), dev.zeros(k, F16)
    dev.cross_entropy(xb, n, 1, wb, k, lb, loss, lse)
    dev.cross_entropy_grad(xb, n, 1, wb, k, lb, lse, dx, dw, gloss=dev.upload_f32(np.ones(n)))
    at = np.concatenate([np.arange(2000), np.arange(n - 2000, n), r.integers(0, n, 20_000)])
    x64, w64 = x[at, None].astype(float), w[:, None].astype(float)
    _, _, p, _ = R.cross_entropy(x64, w64, lab[at], 1.0)
    want, _, g = R.cross_entropy_grad(x64, w64, lab[at], 1.0, p, np.ones(at.size))
    tol = (2.0 ** -11 * 1.01 * np.abs(g) + 2.0 ** -17) @ np.abs(w64) + 2.0 ** -11 * np.abs(want)
    assert np.all(np.abs(dev.read(dx).astype(float)[at, None] - want) <= tol + 2.0 ** -25)
    assert not dev.read(dx)[::1001].any()
    # dw is far beyond f16, with the sign that it has.
    has = lab != NONE
    x64 = x.astype(float)
    dw0 = ((1.0 / (1.0 + np.exp(-2.0 * x64)) - (lab == 0)) * x64 * has).sum()
    assert abs(dw0) > 1e6 and np.array_equal(dev.read(dw), np.sign([dw0, -dw0]) * np.inf)


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
