"""Log probabilities and their gradient at the ends of the logits' range: logits that the scale
brings beyond f32, products with the scale that are large and not exact, rows masked by the
type's lowest value. In rows of one chunk, of several, and in parts."""

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


def _call(dev, z, tokens, name, scale, top):
    """logp, lse, entropy and the list of rows of logits, and the buffers of z, lse and entropy."""
    from emeans_amd import F32, U32
    n, k = z.shape
    p, t = R.Padded(dev, z, name), dev.upload_u32(np.asarray(tokens, np.uint32))
    lp, lse, h = (dev.zeros(n, F32) for _ in range(3))
    ids, tops = dev.zeros(n * top, U32), dev.zeros(n * top, F32)
    dev.log_probs(p.buf, n, k, t, lp, lse, entropy=h, top=top, top_ids=ids if top else None,
                  top_logp=tops if top else None, scale=scale)
    read = [dev.read(b) for b in (lp, lse, h)]
    return (*read, dev.read(ids).reshape(n, top), dev.read(tops).reshape(n, top)), (p, t, lse, h)


def _grad(dev, bufs, scale, gl, gh):
    p, t, lse, h = bufs
    dz = R.Padded(dev, np.zeros_like(p.value), p.name, fill=7.0)
    dev.log_probs_grad(p.buf, p.rows, p.d, t, lse, dz.buf, entropy=h, glogp=dev.upload_f32(gl),
                       gentropy=dev.upload_f32(gh), scale=scale)
    return dz.read()


# Rows of one chunk, of several by four waves, and in parts.
SHAPES = [(6, 40), (1100, 9001), (6, 40001)]


@pytest.mark.parametrize("n,k", SHAPES)
@pytest.mark.parametrize("name,large,scale", [("f32", 3e38, 2.0), ("f32", 2e30, 3e8),
                                              ("bf16", 3e38, 1.5), ("f16", 60000.0, 1e38)])
@pytest.mark.parametrize("top", [0, 5])
def test_a_logit_that_the_scale_makes_infinite(dev, n, k, name, large, scale, top):
    """A product above f32 counts as +infinity: NaN everywhere and no ids, in its row alone."""
    z = np.zeros((n, k))
    z[:, 1] = -1e-6 / scale
    z[0, 0], z[2, k - 1], z[3, [5, k // 2]] = large, large, large
    bad = np.isin(np.arange(n), [0, 2, 3])
    tokens = np.full(n, 3)
    tokens[2], tokens[3] = k - 1, A.NONE
    (lp, lse, h, ids, tops), bufs = _call(dev, z, tokens, name, scale, top)
    assert np.isnan(lse[bad]).all() and np.isnan(h[bad]).all()
    assert np.isnan(lp[[0, 2]]).all() and lp[3] == 0  # (no class was asked for)
    assert (ids[bad] == A.NONE).all() and np.isnan(tops[bad]).all()
    # The others: k classes alike, but one by a millionth.
    tol = 2e-6 + (k / 64 + 96) * U
    assert np.abs(lse[~bad] - np.log(k)).max() <= tol and np.abs(h[~bad] - np.log(k)).max() <= tol
    assert np.abs(lp[~bad] + np.log(k)).max() <= tol
    if top:
        less = bufs[0].value[1, 1] < 0  # (f16 does not hold the millionth)
        assert (ids[~bad] == ([0, 2, 3, 4, 5] if less else [0, 1, 2, 3, 4])).all()
    g = _grad(dev, bufs, scale, np.full(n, 1 / scale), np.full(n, 1 / scale))
    assert np.isnan(g[[0, 2]]).all() and np.isfinite(g[~bad]).all()
