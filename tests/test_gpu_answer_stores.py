"""Results that go through the caches or past them: products whose rows are whole lines, of more
tiles than there are workgroups, and clipped gradients of 128 MB and more."""

import numpy as np
import pytest

from tests import answer_ref as A
from tests import learn_ref as R
from tests import test_gpu_product8 as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from emeans_amd import HipDevice
    d = HipDevice()
    yield d
    d.close()


# Results of 67 and 134 MB, and of 270 MB and more.
@pytest.mark.parametrize("n,d,k", [(16384, 200, 2048), (16385, 100, 2080), (16384, 1, 2048),
                                   (16384, 130, 8320), (8192, 640, 16640), (33000, 128, 4160)])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_products_of_many_whole_tiles(dev, n, d, k, name):
    r = np.random.default_rng(n + d + k)
    (x, xs), (w, ws) = P._codes(r, n, d, False), P._codes(r, k, d, True)
    bx, bw = A.CodeBuf(dev, n, d, x), A.CodeBuf(dev, k, d, w)
    sx, sw = R.Padded(dev, xs, "f32"), R.Padded(dev, ws, "f32")
    y = dev.zeros(n * k, R.kind(name))
    dev.product8(bx.buf, sx.buf, n, d, bw.buf, sw.buf, k, y)
    # Every row of a few tiles, and some of all.
    rows = np.unique(np.r_[0:256, n - 256:n, r.integers(0, n, 400)])
    got = R.decode(dev.read(y).reshape(n, k)[rows], name)
    want, mag, most = P._want(x[rows], xs[rows], w, ws)
    assert np.all(np.abs(got - want) <= P._tol(want, mag, most, d, name))


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("at", [0, 1, 5])
def test_large_gradients_into_outputs(dev, name, at):
    """70 (f32: 36) million elements at an odd address, and short tensors beside them."""
    from emeans_amd import F32, GradNorm
    r = np.random.default_rng(at)
    lengths = [70_000_003 if name == "bf16" else 36_000_001, 1001, 0, 5]
    part = r.standard_normal(1 << 20).astype(np.float32)
    e = 4 if name == "f32" else 2
    raws, grads, outs, held = [], [], [], []
    for n in lengths:
        v = R.encode(np.resize(part, n), name)
        g, o = dev.zeros(n + 16, R.kind(name)), dev.zeros(n + 16, R.kind(name))
        dev.write(g, at, v)
        grads.append(dev.wrap(g.ptr + at * e, n, g.kind))
        outs.append(dev.wrap(o.ptr + (at + 2) * e, n, o.kind))
        raws.append(v)
        held.append((g, o))
    b = dev.zeros(2, F32)
    square = sum((R.decode(v, name) ** 2).sum() for v in raws)
    GradNorm(dev, grads, outs).clip(b, 3.0)
    got = dev.read(b)
    assert abs(got[0] - np.sqrt(square)) <= 2 * R.U32 * np.sqrt(square)
    for v, n, (g, o) in zip(raws, lengths, held):
        want = R.encode(R.decode(v, name).astype(np.float32) * got[1], name)
        whole = dev.read(o)
        assert whole[at + 2:at + 2 + n].tobytes() == want.tobytes()
        assert not whole[:at + 2].any() and not whole[at + 2 + n:].any()
        assert dev.read(g)[at:at + n].tobytes() == v.tobytes()
