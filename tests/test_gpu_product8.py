"""The product of 8-bit codes against 64 bits: from one row to many tiles, depths that end inside
a block, strides and offsets, codes that are not finite."""

import numpy as np
import pytest

from tests import answer_ref as A
from tests import learn_ref as R

pytestmark = pytest.mark.gpu
U = R.U32


@pytest.fixture(scope="module")
def dev():
    from emeans_amd import HipDevice
    d = HipDevice()
    yield d
    d.close()


def _codes(r, rows, d, tall):
    x = r.standard_normal((rows, d)) * np.exp(r.standard_normal((rows, 1)))
    return A.quantize(x, 128 if tall else 1)


def _want(x, xs, w, ws):
    """y in 64 bits, the sum of its terms' magnitudes, and a bound of the largest of each eight
    neighbouring columns' (the product of their largest factors), added."""
    n, d = x.shape
    a = R.f8_decode(x) * A.spread(xs, 1, n, d)
    b = R.f8_decode(w) * A.spread(ws, 128, len(w), d)
    aa, ab = np.abs(a), np.abs(b)
    pad = ((0, 0), (0, -d % 8))
    most = (np.pad(v, pad).reshape(len(v), -1, 8).max(2) for v in (aa, ab))
    return a @ b.T, aa @ ab.T, next(most) @ next(most).T


def _tol(want, mag, most, d, name):
    """A block's 128 products are exact in f32 and added there: at most 128 roundings of the
    partial sums, whatever their order; the scale is a product (two roundings with the sum's),
    and the blocks are added one by one or joined. For 16-bit results the products of eight
    neighbouring columns may be aligned to the largest, with 13 bits below it: seven others
    lose up to 2^-13 of it each."""
    tol = (128 + A.blocks(d) + 8) * U * mag + R.UNIT[name] * np.abs(want) * 1.01 + R.TINY[name]
    return tol if name == "f32" else tol + 7 * 2.0 ** -13 * most


def _run(dev, n, d, k, name, seed, pad=0, off=0):
    r = np.random.default_rng(seed)
    (x, xs), (w, ws) = _codes(r, n, d, False), _codes(r, k, d, True)
    # What lies between the rows is NaN.
    bx, bw = A.CodeBuf(dev, n, d, x, pad, off), A.CodeBuf(dev, k, d, w, 2 * pad, off)
    sx, sw = R.Padded(dev, xs, "f32", pad, off), R.Padded(dev, ws, "f32", 2 * pad, off)
    y = R.Padded(dev, np.zeros((n, k)), name, pad, off, fill=7.0)
    dev.product8(bx.buf, sx.buf, n, d, bw.buf, sw.buf, k, y.buf, ldx=bx.ld, ldxs=sx.ld, ldw=bw.ld,
                 ldws=sw.ld, ldy=y.ld)
    want, mag, most = _want(x, xs, w, ws)
    assert np.all(np.abs(y.read() - want) <= _tol(want, mag, most, d, name))


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 33, 64, 65, 100, 128, 129, 300, 1000])
@pytest.mark.parametrize("d,k", [(128, 128), (300, 1000), (100, 17), (1024, 257), (513, 129)])
def test_sizes(dev, n, d, k):
    name = ["f32", "bf16", "f16"][(n + d + k) % 3]
    pad = (n + k) % 3
    _run(dev, n, d, k, name, n * 7 + d + k, pad, pad)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,d,k", [(1, 1, 1), (3, 16, 2), (5, 31, 1), (2, 127, 300), (700, 129, 900),
                                   (512, 768, 1024), (513, 640, 1025), (40, 5000, 70),
                                   (300, 5008, 300), (2100, 256, 2300)])
def test_types(dev, n, d, k, name):
    _run(dev, n, d, k, name, n + d + k)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,d,k,pad,off", [(1500, 513, 1501, 1, 1), (2000, 100, 2001, 0, 1),
                                           (4001, 77, 5003, 0, 0), (9001, 130, 3001, 2, 0),
                                           (3000, 200, 3004, 0, 2)])
def test_tiles_of_short_blocks_and_more_of_them_than_workgroups(dev, n, d, k, pad, off, name):
    _run(dev, n, d, k, name, n + d, pad, off)


@pytest.mark.parametrize("n,d,k", [(3, 200, 50), (300, 200, 400), (1300, 200, 1400)])
def test_codes_and_scales_that_are_not_finite_stay_in_their_rows(dev, n, d, k):
    r = np.random.default_rng(2)
    (x, xs), (w, ws) = _codes(r, n, d, False), _codes(r, k, d, True)
    x[1, 150], w[7, 3] = 0x7F, 0xFF
    xs[2, 1] = np.inf
    b = [A.CodeBuf(dev, n, d, x), A.CodeBuf(dev, k, d, w)]
    s = [R.Padded(dev, xs, "f32"), R.Padded(dev, ws, "f32")]
    y = R.Padded(dev, np.zeros((n, k)), "f32")
    dev.product8(b[0].buf, s[0].buf, n, d, b[1].buf, s[1].buf, k, y.buf)
    got = y.read()
    assert np.isnan(got[1]).all() and np.isnan(got[:, 7]).all()
    assert not np.isfinite(got[2]).any()
    rows, cols = np.arange(n) > 2, np.arange(k) != 7
    rows[0] = True
    x[1, 150] = w[7, 3] = 0
    xs[2, 1] = 0
    want, mag, most = _want(x, xs, w, ws)
    at = np.ix_(rows, cols)
    assert np.all(np.abs(got[at] - want[at]) <= _tol(want, mag, most, d, "f32")[at])


def test_results_follow_from_the_inputs_alone(dev):
    from emeans_amd import BF16
    r = np.random.default_rng(9)
    n, d, k = 1300, 768, 1000
    (x, xs), (w, ws) = _codes(r, n, d, False), _codes(r, k, d, True)
    b = [A.CodeBuf(dev, n, d, x), A.CodeBuf(dev, k, d, w)]
    s = [R.Padded(dev, xs, "f32"), R.Padded(dev, ws, "f32")]
    y = dev.zeros(n * k, BF16)

    def call():
        dev.product8(b[0].buf, s[0].buf, n, d, b[1].buf, s[1].buf, k, y)
    call()
    first = dev.read(y).tobytes()
    g = A.Graph(dev, call)
    for _ in range(3):
        dev.write(y, 0, np.zeros(n * k, np.uint16))
        g.replay()
        assert dev.read(y).tobytes() == first
        call()
        assert dev.read(y).tobytes() == first
    g.close()


def test_no_rows_and_refusals(dev):
    from emeans_amd import F32, F8, U32, EmeansHipInvalid
    x, w = dev.zeros(10 * 32, F8), dev.zeros(20 * 32, F8)
    s, t, y = dev.zeros(10, F32), dev.zeros(1, F32), dev.zeros(200, F32)
    dev.product8(x, s, 0, 30, w, t, 20, y)
    dev.product8(x, s, 10, 30, w, t, 20, y)
    assert not dev.read(y).any()

    def no(match, *args, **kw):
        with pytest.raises(EmeansHipInvalid, match=match):
            dev.product8(*args, **kw)
    no("d must be", x, s, 10, 0, w, t, 20, y)
    no("k must be", x, s, 10, 30, w, t, 0, y)
    no("x must be an f8", y, s, 10, 30, w, t, 20, y)
    no("w must be an f8", x, s, 10, 30, y, t, 20, y)
    no("xscales must be", x, x, 10, 30, w, t, 20, y)
    no("y must be", x, s, 10, 30, w, t, 20, dev.zeros(200, U32))
    no("x: the buffer's", x, s, 11, 30, w, t, 20, dev.zeros(220, F32))
    no("xscales: the buffer's", dev.zeros(11 * 32, F8), s, 11, 30, w, t, 20, dev.zeros(220, F32))
    no("w: the buffer's", x, s, 10, 30, w, t, 21, dev.zeros(210, F32))
    no("wscales: the buffer's", x, s, 10, 30, dev.zeros(129 * 32, F8), t, 129, dev.zeros(1290, F32))
    no("y: the buffer's", x, s, 10, 30, w, t, 20, dev.zeros(199, F32))
    no("multiple of 16", x, s, 5, 30, w, t, 20, y, ldx=40)
    no("multiple of 16", x, s, 5, 30, w, t, 20, y, ldw=16)
    no("multiple of 16 bytes", dev.wrap(x.ptr + 4, 300, F8), s, 5, 30, w, t, 20, y)
    no("y overlaps x", x, s, 1, 30, w, t, 20, dev.wrap(x.ptr, 20, F32))
    no("y overlaps xscales", x, s, 1, 30, w, t, 10, dev.wrap(s.ptr, 10, F32))
