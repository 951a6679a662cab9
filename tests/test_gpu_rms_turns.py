"""The RMS norm, its codes and its gradient over more rows than its workgroups take at once, so that
each of them takes several in turn: rows on 16 lanes, on a wave and on four waves, with results
of less and of more than 16 MB."""

import numpy as np
import pytest

from tests import learn_ref as R
from tests import test_gpu_rms_norm as T

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from emeans_amd import HipDevice
    d = HipDevice()
    yield d
    d.close()


SIZES = [(40000, 40), (40003, 250), (10007, 300), (9001, 1000), (2500, 2049), (4500, 2000),
         (2500, 4093)]


@pytest.mark.parametrize("rows,d", SIZES + [(1500, 4099)])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_forward_and_gradient(dev, rows, d, name):
    T.test_forward_and_gradient(dev, rows, d, name)


@pytest.mark.parametrize("rows,d", SIZES)
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_codes(dev, rows, d, name):
    T.test_codes(dev, rows, d, name)


@pytest.mark.parametrize("rows,d", SIZES)
@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_in_place(dev, rows, d, name):
    """h in the residual's place and y in x's, dx in dy's: to the bit what they are elsewhere."""
    from emeans_amd import F32
    x, res, w, r = T._inputs(rows, d, rows + d)
    pw, rstd = R.Padded(dev, w[None], "f32"), dev.zeros(rows, F32)
    put = lambda v: R.Padded(dev, v, name)  # noqa: E731
    px, pr, ph, py = put(x), put(res), put(0 * x), put(0 * x)
    dev.rms_norm(px.buf, rows, d, pw.buf, py.buf, residual=pr.buf, h=ph.buf, rstd=rstd)
    dev.rms_norm(px.buf, rows, d, pw.buf, px.buf, residual=pr.buf, h=pr.buf)
    assert np.array_equal(px.read(), py.read()) and np.array_equal(pr.read(), ph.read())
    assert np.array_equal(ph.read(), T._sum(put(x).value, put(res).value, name))
    pd, po = put(r.standard_normal((rows, d))), put(0 * x)
    g = [dev.zeros(d, F32) for _ in range(2)]
    dev.rms_norm_grad(pd.buf, ph.buf, rows, d, pw.buf, rstd, po.buf, g[0])
    dev.rms_norm_grad(pd.buf, ph.buf, rows, d, pw.buf, rstd, pd.buf, g[1])
    assert np.array_equal(pd.read(), po.read()) and po.read().any()
    assert dev.read(g[0]).tobytes() == dev.read(g[1]).tobytes()
