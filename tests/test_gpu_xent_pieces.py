"""The cross entropy's gradients in many pieces of the classes (a workspace that holds the
least of them), the last of one class and more, against 64 bits."""

import numpy as np
import pytest

from tests import learn_ref as R
from tests.test_gpu_cross_entropy import NONE, Run, _inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from emeans_amd import HipDevice
    d = HipDevice()
    d.set_xent_workspace(1)
    yield d
    d.close()


# d = 64: rows as they lie; others are laid out. Few rows and columns: dx in splits.
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,d", [(300, 40), (300, 64), (65, 500), (1000, 200)])
@pytest.mark.parametrize("last", [1, 63, 65, 257])
def test_a_short_last_piece(dev, name, n, d, last):
    k = 2 * 768 + last
    x, w, lab = _inputs(n, d, k, n + d + last)
    lab[:3] = k - 1, 767, 768
    gloss = None if last % 4 == 1 else np.random.default_rng(1).standard_normal(n)
    Run(dev, x, w, lab, name, gloss=gloss).check()


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_one_gradient_alone(dev, name):
    from emeans_amd import F32
    n, d, k = 200, 72, 2 * 768 + 5
    x, w, lab = _inputs(n, d, k, 5)
    both = Run(dev, x, w, lab, name).check()
    xb, wb = R.Padded(dev, x, name), R.Padded(dev, w, name)
    lb, lse = dev.upload_u32(lab), dev.upload_f32(both.lse)
    dx, dw = R.Padded(dev, np.zeros((n, d)), name), R.Padded(dev, np.zeros((k, d)), name)
    dev.cross_entropy_grad(xb.buf, n, d, wb.buf, k, lb, lse, dx.buf, None)
    dev.cross_entropy_grad(xb.buf, n, d, wb.buf, k, lb, lse, None, dw.buf)
    assert np.array_equal(dx.read(), both.dx) and np.array_equal(dw.read(), both.dw)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [40, 64])
@pytest.mark.parametrize("want_dx", [False, True])
def test_a_row_without_a_label_that_is_not_finite(dev, name, d, want_dx):
    """Found with the first piece, and kept out of dw in the others."""
    from emeans_amd import F32
    n, k = 300, 2 * 768 + 1
    x, w, lab = _inputs(n, d, k, d)
    lab[[2, 299]] = NONE
    w[::3, 17] = 0.0
    clean = Run(dev, x, w, lab, name).check()
    y = x.copy()
    y[2, 17], y[299] = np.nan, np.inf
    px, pw, lb = R.Padded(dev, y, name), R.Padded(dev, w, name), dev.upload_u32(lab)
    loss, lse = dev.zeros(n, F32), dev.zeros(n, F32)
    dx, dw = dev.zeros(n * d, R.kind(name)), dev.zeros(k * d, R.kind(name))
    dev.cross_entropy(px.buf, n, d, pw.buf, k, lb, loss, lse)
    dev.cross_entropy_grad(px.buf, n, d, pw.buf, k, lb, lse, dx if want_dx else None, dw)
    assert np.array_equal(R.decode(dev.read(dw), name).reshape(k, d), clean.dw)
    if want_dx:
        assert np.array_equal(R.decode(dev.read(dx), name).reshape(n, d), clean.dx)
