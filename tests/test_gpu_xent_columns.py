"""float32 cross entropy of columns of unequal sizes, which the classes make up for: each
element is held to 2^-22 of itself, or 2^-49 of its row's largest."""

import numpy as np
import pytest

from tests import learn_ref as R
from tests.test_gpu_cross_entropy import NONE, U, Run, _inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from emeans_amd import HipDevice
    d = HipDevice()
    yield d
    d.close()


# Of a product of two elements: both held to 2^-22, the product of what is left out of both
# another 2^-22 (2^-20 for all three); or, for the smallest of a row, 2^-49 of its largest
# times the other (three times that: 2^-47).
REL, LOW = 2.0 ** -20, 2.0 ** -47


def check(run):
    x, w, lab, s = run.x, run.w, run.lab, abs(run.scale)
    n, d = x.shape
    k = w.shape[0]
    has = lab != NONE
    up = np.where(has, 1.0 / max(1, has.sum()), 0)
    loss, lse, p, z = R.cross_entropy(x, w, lab, run.scale)
    ax, aw = np.abs(x), np.abs(w)
    ez = s * (((d + 16) * U + REL) * (ax @ aw.T)
              + LOW * (ax.max(1)[:, None] * aw.sum(1)[None] + ax.sum(1)[:, None] * aw.max(1)[None]))
    ez = ez + 8 * U * np.abs(z)
    el = (p * ez).sum(1) * 1.01 + (k / 16 + 64) * U + 8 * U * np.abs(lse) + 4 * U * np.abs(z).max(1)
    assert np.all(np.abs(run.lse - lse) <= el)
    at = np.where(has, lab, 0).astype(np.int64)
    tol = np.where(has, el + ez[np.arange(n), at] + 4 * U * np.abs(loss), 0.0)
    assert np.all(np.abs(run.loss - loss) <= tol)
    dx, dw, g = R.cross_entropy_grad(x, w, lab, run.scale, p, up)
    sg, top = (s * up)[:, None], s * up.max()
    eg = sg * p * ((ez + el[:, None]) * 1.01 + 8 * U * (np.abs(z) + np.abs(lse)[:, None]))
    eg = eg + REL * np.abs(g) + 4 * U * sg * has[:, None] + 2.0 ** -40 * top
    eg[~has] = 0.0
    ag, hx = np.abs(g), np.where(has[:, None], ax, 0.0)
    tol = eg @ aw + ((k + 64) * U + REL) * (ag @ aw) + LOW * (ag @ aw.max(1))[:, None]
    assert np.all(np.abs(run.dx - dx) <= tol + U * np.abs(dx))
    tol = eg.T @ hx + ((n + 64) * U + REL) * (ag.T @ hx) + LOW * (ag.T @ hx.max(1))[:, None]
    assert np.all(np.abs(run.dw - dw) <= tol + U * np.abs(dw))


# Few rows, one and three passes over the planes, tiles of every shape, splits of them that
# end before, at and after the last pass begins.
SIZES = [(64, 64, 200), (65, 64, 200), (300, 64, 200), (150, 21, 671), (658, 16, 20),
         (9944, 16, 390), (9181, 16, 910), (2500, 70, 1250), (6679, 536, 712), (8456, 142, 1820),
         (5521, 17, 2207)]


@pytest.mark.parametrize("size", [1e3, 1e4, 1e5])
@pytest.mark.parametrize("n,d,k", SIZES)
def test_columns_that_the_classes_make_up_for(dev, n, d, k, size):
    x, w, lab = _inputs(n, d, k, n + d)
    c = np.where(np.arange(d) % 2, size, 1 / size)
    check(Run(dev, x * c, w / c, lab, "f32"))


@pytest.mark.parametrize("n,d,k", [(300, 64, 200), (2500, 70, 1250)])
def test_columns_over_ten_decades(dev, n, d, k):
    x, w, lab = _inputs(n, d, k, n + d)
    c = 10.0 ** np.linspace(-5, 5, d)
    check(Run(dev, x * c, w / c, lab, "f32", scale=0.5))
    check(Run(dev, x / c, w * c * 1e-6, lab, "f32", scale=1e6))


def test_few_and_more_rows_agree(dev):
    """64 rows go another way than 65."""
    x, w, lab = _inputs(65, 64, 200, 7)
    c = np.where(np.arange(64) % 2, 1e4, 1e-4)
    more, few = Run(dev, x * c, w / c, lab, "f32"), Run(dev, x[:64] * c, w / c, lab[:64], "f32")
    # Sums of 64 terms of about 1 / 8 each, in f32 in two orders: 64 roundings of 1.
    assert np.abs(more.lse[:64] - few.lse).max() <= 64 * U * np.abs(few.lse).max()
