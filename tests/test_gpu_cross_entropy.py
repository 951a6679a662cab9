"""Softmax cross entropy and its gradients against 64 bits: one row to
thousands, one class to tens of thousands, every element type, strides, offsets, rows without a label,
rows and classes whose values are not finite, and what the calls refuse."""

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


def _inputs(n, d, k, seed, none=0.1):
    r = np.random.default_rng(seed)
    w = r.standard_normal((k, d)) / np.sqrt(d)
    lab = r.integers(0, k, n).astype(np.uint32)
    x = r.standard_normal((n, d)) + w[lab] * (4 * r.random((n, 1)))
    lab[r.random(n) < none] = NONE
    return x, w, lab


class Run:
    def __init__(self, dev, x, w, lab, name, scale=1.0, pad=0, off=0, gloss=None, grad=True):
        from emeans_amd import F32
        n, d = x.shape
        k = w.shape[0]
        self.name, self.scale, self.lab, self.gloss = name, scale, lab, gloss
        px, pw = R.Padded(dev, x, name, pad, off), R.Padded(dev, w, name, 2 * pad, off)
        self.x, self.w = px.value, pw.value
        lb = dev.upload_u32(lab)
        loss, lse = dev.upload_f32(np.full(n, 9.0)), dev.upload_f32(np.full(n, 9.0))
        dev.cross_entropy(px.buf, n, d, pw.buf, k, lb, loss, lse, scale=scale, ldx=px.ld,
                          ldw=pw.ld)
        self.loss, self.lse = dev.read(loss).astype(float), dev.read(lse).astype(float)
        if not grad:
            return
        dx = R.Padded(dev, np.zeros((n, d)), name, 3 * pad, off, fill=7.0)
        dw = R.Padded(dev, np.zeros((k, d)), name, pad, off, fill=7.0)
        up = None if gloss is None else dev.upload_f32(gloss)
        dev.cross_entropy_grad(px.buf, n, d, pw.buf, k, lb, lse, dx.buf, dw.buf, gloss=up,
                               scale=scale, ldx=px.ld, ldw=pw.ld, lddx=dx.ld, lddw=dw.ld)
        self.dx, self.dw = dx.read(), dw.read()

    def check(self):
        """Products of d terms in f32, of operands held to 2^-22 of each: a
        logit is within E = scale ((d + 16) u + 2^-20) sum |x w| (+ what a row's
        smallest elements lose next to its largest, 2^-37 of it). The rest of
        the softmax: roundings of exponents (u |z|) and a sum's chain."""
        x, w, lab = self.x, self.w, self.lab
        n, d = x.shape
        k = w.shape[0]
        has = lab != NONE
        up = np.where(has, 1.0 / max(1, has.sum()), 0) if self.gloss is None else \
            np.float32(self.gloss).astype(float)
        loss, lse, p, z = R.cross_entropy(x, w, lab, self.scale)
        s = abs(self.scale)
        ez = s * (((d + 16) * U + 2.0 ** -20) * (np.abs(x) @ np.abs(w).T)
                  + 2.0 ** -37 * d * np.abs(x).max(1)[:, None] * np.abs(w).max(1)[None, :])
        ez = ez + 8 * U * np.abs(z)
        el = (p * ez).sum(1) * 1.01 + (k / 16 + 64) * U + 8 * U * np.abs(lse) + 4 * U * np.abs(z).max(1)
        assert np.all(np.abs(self.lse - lse) <= el)
        at = np.where(has, lab, 0).astype(np.int64)
        tol = np.where(has, el + ez[np.arange(n), at] + 4 * U * np.abs(loss), 0.0)
        assert np.all(np.abs(self.loss - loss) <= tol)
        if not hasattr(self, "dx"):
            return self
        dx, dw, g = R.cross_entropy_grad(x, w, lab, self.scale, p, up)
        unit = {"f32": 2.0 ** -20, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[self.name]
        top = s * np.abs(np.where(has, up, 0)).max()
        sg = (s * np.abs(np.where(has, up, 0)))[:, None]
        eg = sg * p * ((ez + el[:, None]) * 1.01 + 8 * U * (np.abs(z) + np.abs(lse)[:, None]))
        eg = eg + unit * np.abs(g) * 1.01 + 4 * U * sg * has[:, None] + 2.0 ** -36 * top
        eg[~has] = 0.0
        hx = np.where(has[:, None], np.abs(x), 0.0)
        out = R.UNIT[self.name]
        tol = eg @ np.abs(w) + ((k + 64) * U + 2.0 ** -20) * (np.abs(g) @ np.abs(w))
        assert np.all(np.abs(self.dx - dx) <= tol + out * 1.01 * np.abs(dx) + R.TINY[self.name])
        tol = eg.T @ hx + ((n + 64) * U + 2.0 ** -20) * (np.abs(g).T @ hx)
        assert np.all(np.abs(self.dw - dw) <= tol + out * 1.01 * np.abs(dw) + R.TINY[self.name])
        assert not self.dx[~has].any()
        return self


SIZES = [(1, 1, 1), (1, 1, 2), (2, 3, 5), (16, 384, 256), (1, 768, 1000), (5, 64, 64),
         (65, 33, 129), (300, 100, 37), (257, 300, 1000), (256, 32, 256), (64, 1024, 300),
         (513, 48, 515), (40, 7, 3000), (3000, 20, 10), (1000, 256, 3), (33, 65, 64),
         (17, 2100, 40), (1200, 128, 1500)]


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,d,k", SIZES)
def test_against_64_bits(dev, n, d, k, name):
    x, w, lab = _inputs(n, d, k, n + d + k)
    gloss = None if (n + k) % 2 else np.random.default_rng(1).standard_normal(n)
    Run(dev, x, w, lab, name, gloss=gloss).check()


# Enough rows, columns or classes for each of the products' tile shapes, and for
# sums split over the depth, at sizes that end inside a tile.
TILES = [(10_007, 300, 1000), (2100, 770, 1250), (4097, 190, 385), (700, 64, 4500), (5000, 384, 130)]


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,d,k", TILES)
def test_every_tile_shape(dev, n, d, k, name):
    x, w, lab = _inputs(n, d, k, n + d + k)
    Run(dev, x, w, lab, name).check()


@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("n,k,want_dx", [(300, 140, False), (300, 140, True), (4000, 700, False),
                                         (33_000, 65, True), (33_000, 65, False)])
def test_rows_without_a_label_keep_out_of_dw(dev, name, value, n, k, want_dx):
    """One value of such a row that is not finite, where some classes have a zero, at
    few rows and at more than are counted on the way; with dx and without."""
    from emeans_amd import F32
    d = 64
    x, w, lab = _inputs(n, d, k, n + k)
    lab[[3, n // 2, n - 1]] = NONE
    w[::3, 17] = 0.0
    clean = R.Padded(dev, x, name).value
    y = x.copy()
    y[3, 17], y[n // 2, 17], y[n - 1, 17] = value, value, value
    px, pw, lb = R.Padded(dev, y, name), R.Padded(dev, w, name), dev.upload_u32(lab)
    loss, lse = dev.zeros(n, F32), dev.zeros(n, F32)
    dx, dw = dev.zeros(n * d, R.kind(name)), dev.zeros(k * d, R.kind(name))
    dev.cross_entropy(px.buf, n, d, pw.buf, k, lb, loss, lse)
    dev.cross_entropy_grad(px.buf, n, d, pw.buf, k, lb, lse, dx if want_dx else None, dw)
    got = R.decode(dev.read(dw), name).reshape(k, d)
    has = lab != NONE
    _, lse64, p, z = R.cross_entropy(clean, pw.value, lab, 1.0)
    up = np.where(has, 1.0 / has.sum(), 0.0)
    _, want, g = R.cross_entropy_grad(clean, pw.value, lab, 1.0, p, up)
    # (The bounds of Run.check, coarser: a logit within 2^-15 of its terms' sizes.)
    ez = 2.0 ** -15 * (np.abs(clean) @ np.abs(pw.value).T + np.abs(lse64)[:, None] + 1)
    unit = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}[name]
    eg = up[:, None] * p * ez + 1.01 * unit * np.abs(g) + 2.0 ** -36 * up.max()
    eg[~has] = 0.0
    tol = eg.T @ np.abs(clean) + (n + 64) * U * (np.abs(g).T @ np.abs(clean))
    assert np.all(np.abs(got - want) <= tol + 1.01 * R.UNIT[name] * np.abs(want) + R.TINY[name])
    if want_dx:
        assert not R.decode(dev.read(dx), name).reshape(n, d)[~has].any()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [5, 300, 40_000])
def test_a_wrong_label_is_an_error_of_the_gradient_too(dev, name, n):
    from emeans_amd import EmeansHipInvalid, F32
    x, w, lab = _inputs(n, 16, 9, n)
    px, pw = R.Padded(dev, x, name), R.Padded(dev, w, name)
    loss, lse = dev.zeros(n, F32), dev.zeros(n, F32)
    dx, dw = dev.zeros(n * 16, R.kind(name)), dev.zeros(9 * 16, R.kind(name))
    dev.cross_entropy(px.buf, n, 16, pw.buf, 9, dev.upload_u32(lab), loss, lse)
    dev.sync()
    bad = lab.copy()
    bad[n - 2] = 9
    dev.cross_entropy_grad(px.buf, n, 16, pw.buf, 9, dev.upload_u32(bad), lse, dx, dw)
    with pytest.raises(EmeansHipInvalid, match="label out of range"):
        dev.sync()
    dev.cross_entropy_grad(px.buf, n, 16, pw.buf, 9, dev.upload_u32(lab), lse, dx, dw)
    dev.sync()


# 16-bit rows and classes at every alignment that an element may have, at either side of
# the last vector's end.
@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("d", [8, 31, 32, 33, 39, 41, 65, 127])
@pytest.mark.parametrize("pad,off", [(0, 0), (0, 1), (1, 2), (1, 3)])
def test_few_rows_at_any_alignment(dev, name, d, pad, off):
    x, w, lab = _inputs(11 + 3 * d % 50, d, 83, d)
    Run(dev, x, w, lab, name, pad=pad, off=off, grad=False).check()


# Few rows, so many classes that several are taken together, at either side of the
# sizes where they are.
FEW = [(1, 40, 65_537), (4, 37, 65_536), (4, 33, 65_535), (5, 64, 16_384), (5, 64, 16_383),
       (16, 33, 20_001), (30, 48, 17_001), (50, 20, 16_999), (64, 64, 16_401)]


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,d,k", FEW)
def test_few_rows_many_classes(dev, n, d, k, name):
    x, w, lab = _inputs(n, d, k, n + d + k)
    lab[0] = k - 1
    Run(dev, x, w, lab, name, scale=1.5, pad=n % 2, off=d % 2, grad=False).check()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,d,k", [(9, 40, 70), (270, 64, 300), (100, 33, 513)])
@pytest.mark.parametrize("pad,off", [(0, 1), (3, 0), (8, 5)])
def test_strides_and_offsets(dev, name, n, d, k, pad, off):
    x, w, lab = _inputs(n, d, k, pad + n)
    Run(dev, x, w, lab, name, pad=pad, off=off).check()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [0.0, -3.0, 20.0])
def test_scale_and_unit_rows(dev, name, scale):
    x, w, lab = _inputs(200, 96, 150, 4)
    x /= np.linalg.norm(x, axis=1, keepdims=True)
    w /= np.linalg.norm(w, axis=1, keepdims=True)
    Run(dev, x, w, lab, name, scale=scale).check()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", [1e-4, 30.0])
def test_flat_and_settled_rows(dev, name, size):
    """Logits that hardly differ, and logits of thousands, where all but one
    class underflow."""
    x, w, lab = _inputs(130, 80, 90, 8)
    Run(dev, x * size, w * size, lab, name).check()


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_no_row_has_a_label(dev, name):
    x, w, _ = _inputs(70, 50, 60, 6)
    r = Run(dev, x, w, np.full(70, NONE, np.uint32), name).check()
    assert not r.loss.any() and not r.dx.any() and not r.dw.any()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [20, 300])
def test_rows_that_are_not_finite(dev, name, n):
    """A row without a label may hold anything; a labelled one with a NaN has a
    loss and gradient of NaN and spoils no other row's."""
    x, w, lab = _inputs(n, 70, 90, 9)
    lab[3], lab[5], lab[7] = NONE, NONE, 2
    clean = Run(dev, x, w, lab, name).check()
    y = x.copy()
    y[3, 10], y[5] = np.nan, np.inf
    r = Run(dev, y, w, lab, name)
    rest = np.ones(n, bool)
    rest[[3, 5]] = False
    assert np.array_equal(r.loss, clean.loss) and np.array_equal(r.lse[rest], clean.lse[rest])
    assert np.array_equal(r.dx, clean.dx) and np.array_equal(r.dw, clean.dw)
    y[7, 0] = np.nan
    r = Run(dev, y, w, lab, name)
    rest[7] = False
    assert np.isnan(r.loss[7]) and np.isnan(r.dx[7]).all()
    assert np.array_equal(r.loss[rest], clean.loss[rest])
    assert np.array_equal(r.dx[rest], clean.dx[rest])


def test_a_class_that_is_not_finite_spoils_every_row(dev):
    x, w, lab = _inputs(20, 64, 70, 2)
    w[11, 3] = np.nan
    r = Run(dev, x, w, lab, "f32", grad=False)
    assert np.isnan(r.lse).all() and np.isnan(r.loss[lab != NONE]).all()


def test_wide_ranges_in_one_matrix(dev):
    """float32 rows and classes over thirty decades: each is held to its own size."""
    x, w, lab = _inputs(150, 64, 100, 12)
    x *= 10.0 ** np.linspace(-18, 12, 150)[:, None]
    w *= 10.0 ** np.linspace(-12, -10, 100)[:, None]
    Run(dev, x, w, lab, "f32").check()


@pytest.mark.parametrize("n", [150, 3000])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_zero_rows_and_classes(dev, name, n):
    """A row or a class of zeros (a cluster that was never used) has no size of its own
    to be held to, and takes none of the others' precision."""
    x, w, lab = _inputs(n, 64, 300, 12)
    x[5], w[7], w[200:] = 0.0, 0.0, 0.0
    Run(dev, x, w, lab, name).check()
    Run(dev, 0 * x, w, lab, name).check()
    Run(dev, x, 0 * w, lab, name).check()


@pytest.mark.parametrize("n", [150, 3000])
def test_a_few_rows_and_classes_of_another_size(dev, n):
    """float32 rows and classes nearly of one size, and some of a thousandth of it or a thousand
    times it."""
    x, w, lab = _inputs(n, 64, 300, 13)
    Run(dev, x, w, lab, "f32").check()
    y, v = x.copy(), w.copy()
    y[::7] *= 1e-3
    Run(dev, y, w, lab, "f32").check()
    v[::9] *= 1e-3
    Run(dev, x, v, lab, "f32", gloss=np.random.default_rng(2).standard_normal(n)).check()
    v[3] *= 1e3
    Run(dev, y, v, lab, "f32").check()


def test_labels_out_of_range_are_reported(dev):
    from emeans_amd import EmeansHipInvalid, F32
    x, w, lab = _inputs(50, 40, 30, 3, none=0.0)
    ok = Run(dev, x, w, lab, "f32").check()
    bad = lab.copy()
    bad[4] = 30
    xb, wb, lb = dev.upload_f32(x), dev.upload_f32(w), dev.upload_u32(bad)
    loss, lse, dx, dw = dev.zeros(50, F32), dev.zeros(50, F32), dev.zeros(2000, F32), dev.zeros(1200, F32)
    dev.cross_entropy(xb, 50, 40, wb, 30, lb, loss, lse)
    with pytest.raises(EmeansHipInvalid, match="label out of range"):
        dev.sync()
    dev.sync()
    assert dev.read(loss)[4] == 0.0
    assert np.array_equal(np.delete(dev.read(loss), 4), np.delete(ok.loss, 4).astype(np.float32))
    dev.cross_entropy_grad(xb, 50, 40, wb, 30, lb, lse, dx, dw)
    with pytest.raises(EmeansHipInvalid, match="label out of range"):
        dev.read(dx)
    assert not dev.read(dx).reshape(50, 40)[4].any()


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_one_gradient_alone(dev, name):
    from emeans_amd import F32
    for n, d, k in ((30, 40, 50), (300, 64, 700)):
        x, w, lab = _inputs(n, d, k, 5)
        both = Run(dev, x, w, lab, name)
        xb, wb = R.Padded(dev, x, name), R.Padded(dev, w, name)
        lb, lse = dev.upload_u32(lab), dev.upload_f32(both.lse)
        dx, dw = R.Padded(dev, np.zeros((n, d)), name), R.Padded(dev, np.zeros((k, d)), name)
        dev.cross_entropy_grad(xb.buf, n, d, wb.buf, k, lb, lse, dx.buf, None)
        dev.cross_entropy_grad(xb.buf, n, d, wb.buf, k, lb, lse, None, dw.buf)
        assert np.array_equal(dx.read(), both.dx) and np.array_equal(dw.read(), both.dw)
        loss = dev.zeros(n, F32)
        dev.cross_entropy(xb.buf, n, d, wb.buf, k, lb, loss)
        assert np.array_equal(dev.read(loss), both.loss.astype(np.float32))


def test_gradient_is_the_difference(dev):
    """Along random directions, against central differences of the 64-bit mean
    loss: h^2 and 1e-16 / h leave 1e-9 of the terms, the f32 gradient 2e-5."""
    n, d, k, h = 40, 60, 33, 1e-5
    x, w, lab = _inputs(n, d, k, 21)
    r = Run(dev, x, w, lab, "f32", scale=1.5).check()
    has = lab != NONE
    rng = np.random.default_rng(6)

    def mean(x, w):
        return R.cross_entropy(x, w, lab, 1.5)[0].sum() / has.sum()

    for _ in range(3):
        ex, ew = rng.standard_normal((n, d)), rng.standard_normal((k, d))
        for grad, e, at in ((r.dx, ex, 0), (r.dw, ew, 1)):
            up, down = [r.x, r.w], [r.x, r.w]
            up[at], down[at] = up[at] + h * e, down[at] - h * e
            diff = (mean(*up) - mean(*down)) / (2 * h)
            assert abs((grad * e).sum() - diff) <= 2e-5 * np.abs(grad * e).sum()


def test_no_rows(dev):
    from emeans_amd import F32, U32
    e, w, u = dev.zeros(0, F32), dev.upload_f32(np.ones(12)), dev.zeros(0, U32)
    dev.cross_entropy(e, 0, 4, w, 3, u, e)
    dw = dev.upload_f32(np.ones(12))
    dev.cross_entropy_grad(e, 0, 4, w, 3, u, e, e, dw)
    assert not dev.read(dw).any()


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_the_same_bits_every_time(dev, name):
    x, w, lab = _inputs(700, 100, 900, 2)
    a, b = (Run(dev, x, w, lab, name) for _ in range(2))
    for what in ("loss", "lse", "dx", "dw"):
        assert np.array_equal(getattr(a, what), getattr(b, what))


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_many_rows_and_classes_by_sample(dev, name):
    """Large enough for several pieces of the classes: rows and classes picked at
    random, each from its definition."""
    from emeans_amd import F32
    n, d, k = 9001, 40, 70_001
    x, w, lab = _inputs(n, d, k, 31)
    lab[np.flatnonzero(lab != NONE)[:20]] = k - 1
    px, pw, lb = R.Padded(dev, x, name), R.Padded(dev, w, name), dev.upload_u32(lab)
    loss, lse = dev.zeros(n, F32), dev.zeros(n, F32)
    dx, dw = dev.zeros(n * d, R.kind(name)), dev.zeros(k * d, R.kind(name))
    dev.cross_entropy(px.buf, n, d, pw.buf, k, lb, loss, lse)
    dev.cross_entropy_grad(px.buf, n, d, pw.buf, k, lb, lse, dx, dw)
    loss, lse = dev.read(loss).astype(float), dev.read(lse).astype(float)
    dx = R.decode(dev.read(dx), name).reshape(n, d)
    dw = R.decode(dev.read(dw), name).reshape(k, d)
    x, w, has = px.value, pw.value, lab != NONE
    unit = {"f32": 2.0 ** -19, "f16": 2.0 ** -10.5, "bf16": 2.0 ** -7.5}[name]
    r = np.random.default_rng(7)
    rows = np.concatenate([[0, n - 1], r.integers(0, n, 30)])
    l64, s64, p, _ = R.cross_entropy(x[rows], w, lab[rows], 1.0)
    assert np.all(np.abs(lse[rows] - s64) <= 2e-5) and np.all(np.abs(loss[rows] - l64) <= 3e-5)
    up = np.full(len(rows), 1.0 / has.sum())
    want, _, g = R.cross_entropy_grad(x[rows], w, lab[rows], 1.0, p, up)
    # (Each g is within its type's unit and 1e-4 relative of the softmax's own error.)
    tol = (unit + 1e-4) * (np.abs(g) @ np.abs(w)) + unit * np.abs(want) + R.TINY[name]
    assert np.all(np.abs(dx[rows] - want) <= tol)
    cols = np.unique(np.concatenate([[0, k - 1, 65535, 65536], r.integers(0, k, 60),
                                     lab[has][:20].astype(int)]))
    z = x @ w[cols].T
    g = np.exp(z - lse[:, None]) - (lab[:, None] == cols[None, :])
    g = g * (has / has.sum())[:, None]
    want = g.T @ x
    top = 1.0 / has.sum()
    tol = (unit + 1e-4) * (np.abs(g).T @ np.abs(x)) + 2.0 ** -36 * top * np.abs(x).sum(0)
    assert np.all(np.abs(dw[cols] - want) <= tol + unit * np.abs(want) + R.TINY[name])


def test_refusals(dev):
    from emeans_amd import BF16, F16, F32, F8, U32, EmeansHipInvalid
    z = dev.zeros
    x, w, lab, loss, lse = z(60, F32), z(80, F32), z(6, U32), z(6, F32), z(6, F32)
    ok = (x, 6, 10, w, 8, lab, loss, lse)
    dev.cross_entropy(*ok)

    def refused(fn, *a, **k):
        with pytest.raises(EmeansHipInvalid):
            fn(*a, **k)

    def but(i, b):
        return ok[:i] + (b,) + ok[i + 1:]

    f = dev.cross_entropy
    refused(f, *but(2, 0))
    refused(f, *but(4, 0))
    refused(f, *but(4, 9))
    refused(f, *but(1, 7))
    refused(f, *but(0, z(60, BF16)))                 # one kind for both
    refused(f, *but(0, z(60, F8)))
    refused(f, *but(0, z(60, U32)))
    refused(f, *but(5, z(6, F32)))
    refused(f, *but(5, z(5, U32)))
    refused(f, *but(6, z(6, F16)))
    refused(f, *but(6, z(5, F32)))
    refused(f, *but(6, x))                           # overlaps
    refused(f, *but(7, loss))
    refused(f, *ok, ldx=9)
    refused(f, *ok, ldw=11)
    refused(f, *ok, scale=float("inf"))
    refused(f, *but(0, dev.wrap(x.ptr + 2, 60, F32)))
    g = dev.cross_entropy_grad
    dx, dw = z(60, F32), z(80, F32)
    ok = (x, 6, 10, w, 8, lab, lse, dx, dw)
    g(*ok)
    refused(g, *but(7, z(60, BF16)))
    refused(g, *but(8, z(79, F32)))
    refused(g, *but(7, x))
    refused(g, *but(8, w))
    refused(g, *but(7, dw))
    refused(g, *but(6, z(5, F32)))
    refused(g, *ok, gloss=z(5, F32))
    refused(g, *ok, gloss=z(6, F16))
    refused(g, *ok, lddw=9)
