"""Products of 8-bit codes that do not average out: all positive, sizes spread over many powers of
two, so that what the 8-bit matrix cores cut has one sign; by few rows and by tiles."""

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


@pytest.mark.parametrize("n,d,k", [(1, 1024, 700), (16, 300, 513), (64, 1000, 300), (700, 1024, 900),
                                   (2100, 640, 2300)])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("spread", [1.0, 2.0, 4.0])
def test_positive_codes(dev, n, d, k, name, spread):
    """f32 results: the products are exact, 128 roundings of a block's partial sums and a few more.
    16-bit ones: of each eight neighbours seven may lose 2^-13 of the largest, which is at most
    the product of the largest factors, and the result is rounded once."""
    r = np.random.default_rng(n + d)
    x, w = (np.exp(spread * r.standard_normal((m, d))) for m in (n, k))
    x *= 0.01 / x.mean()
    w *= 0.01 / w.mean()
    (x, xs), (w, ws) = A.quantize(x, 1), A.quantize(w, 128)
    bx, bw = A.CodeBuf(dev, n, d, x), A.CodeBuf(dev, k, d, w)
    sx, sw = R.Padded(dev, xs, "f32"), R.Padded(dev, ws, "f32")
    y = R.Padded(dev, np.zeros((n, k)), name, fill=7.0)
    dev.product8(bx.buf, sx.buf, n, d, bw.buf, sw.buf, k, y.buf)
    a = R.f8_decode(x) * A.spread(xs, 1, n, d)
    b = R.f8_decode(w) * A.spread(ws, 128, k, d)
    want = a @ b.T
    tol = (128 + A.blocks(d) + 8) * U * want + R.UNIT[name] * want + R.TINY[name]
    if name != "f32":
        pad = ((0, 0), (0, -d % 8))
        p, q = (np.pad(v, pad).reshape(len(v), -1, 8).max(2) for v in (a, b))
        tol = tol + 7 * 2.0 ** -13 * (p @ q.T)
    got = y.read()
    if name == "f16":  # (one sum of the widest codes is 217,688)
        over = want > 1.01 * 65504
        assert over.sum() <= 1 and np.isposinf(got[over]).all()
        got, want, tol = got[~over], want[~over], tol[~over]
    assert (want > 0).all() and np.all(np.abs(got - want) <= tol)
