"""The cross entropy's gradients in many pieces of the classes and blocks of the rows (a small
workspace), the last of one class and more, against 64 bits."""

import numpy as np
import pytest

from tests import learn_ref as R
from tests.test_gpu_cross_entropy import NONE, Run, _inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from emeans_amd import HipDevice
    d = HipDevice()
    yield d
    d.close()


def _small(dev, n, name, blocks):
    """Pieces of 768 classes of all rows, or blocks of 256 rows, too."""
    planes = 4 if name == "f32" else 1
    dev.set_xent_workspace(1 if blocks else -(-n // 256) * 256 * 768 * 2 * planes)


# d = 64: rows as they lie; others are laid out. Few rows and columns: dx in splits.
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,d", [(300, 40), (300, 64), (65, 500), (1000, 200), (513, 64)])
@pytest.mark.parametrize("last", [1, 63, 65, 257])
@pytest.mark.parametrize("blocks", [False, True])
def test_a_short_last_piece(dev, name, n, d, last, blocks):
    _small(dev, n, name, blocks)
    k = 2 * 768 + last
    x, w, lab = _inputs(n, d, k, n + d + last)
    lab[:3] = k - 1, 767, 768
    gloss = None if last % 4 == 1 else np.random.default_rng(1).standard_normal(n)
    Run(dev, x, w, lab, name, gloss=gloss).check()


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("n,k", [(300, 40), (1025, 1000)])
def test_blocks_of_rows_alone(dev, name, n, k):
    """All classes in one piece or two: dx as it comes, dw a sum over the blocks."""
    _small(dev, n, name, True)
    x, w, lab = _inputs(n, 50, k, n)
    Run(dev, x, w, lab, name, pad=3).check()


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("blocks", [False, True])
def test_one_gradient_alone(dev, name, blocks):
    from emeans_amd import F32
    n, d, k = 300, 72, 2 * 768 + 5
    _small(dev, n, name, blocks)
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
@pytest.mark.parametrize("blocks", [False, True])
def test_a_row_without_a_label_that_is_not_finite(dev, name, d, want_dx, blocks):
    """Found with the first piece, and kept out of dw in the others."""
    from emeans_amd import F32
    n, k = 300, 2 * 768 + 1
    _small(dev, n, name, blocks)
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
