"""ClusterHead in half precision at a full batch: the gradients of a mean over many rows,
most of them settled, keep their bits. And the gradients' loss scale by itself."""

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


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
def test_gradients_of_a_full_batch(dev, kind):
    from emeans_amd.head import ClusterHead
    n, d, k = 16384, 96, 1000
    r = np.random.default_rng(8)
    w = r.standard_normal((k, d)) / np.sqrt(d)
    lab = np.minimum(r.zipf(1.3, n) - 1, k - 1).astype(np.int32)  # (most classes are rare)
    x = w[lab] * (30 * r.random((n, 1))) + 0.3 * r.standard_normal((n, d))
    lab[::50] = -1
    head = ClusterHead(d, k, kind=R.kind(kind), centroids=2 * w, dev=dev)
    xb, lb = head.rows(x), head.labels(lab)
    raw_w = dev.read(head._w)
    dev.read_f32(head.step(xb, lb, n, 1e-3))
    y = R.decode(dev.read(head._y), kind).reshape(-1, d)[:n]
    w64 = R.decode(raw_w, kind).reshape(k, d)
    got_dy = R.decode(dev.read(head._dy), kind).reshape(-1, d)[:n] / head.loss_scale
    got_dw = R.decode(dev.read(head._dw), kind).reshape(k, d) / head.loss_scale
    lab = np.where(lab < 0, NONE, lab).astype(np.uint32)
    has = lab != NONE
    up = np.where(has, 1.0 / has.sum(), 0.0)
    _, lse, p, z = R.cross_entropy(y, w64, lab, 1.0)
    dy, dw, g = R.cross_entropy_grad(y, w64, lab, 1.0, p, up)
    # A logit of 96 terms and its exponential: within 2^-15 of the terms' sizes; G: its
    # type's unit; the result: another, and its least number over a thousand (a few bits of a
    # gradient of a settled row: 1 / 16,384 of a class's weights times a hundredth).
    unit = {"f32": 2.0 ** -20, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[kind]
    ez = 2.0 ** -15 * (np.abs(y) @ np.abs(w64).T / np.sqrt(d) + np.abs(lse)[:, None] + 1)
    eg = up[:, None] * p * ez + 1.01 * unit * np.abs(g) + 4 * U * up[:, None] + 2.0 ** -36 * up.max()
    eg[~has] = 0.0
    out, tiny = R.UNIT[kind], R.TINY[kind] / 1024
    tol = eg @ np.abs(w64) + (k + 64) * U * (np.abs(g) @ np.abs(w64))
    assert np.all(np.abs(got_dy - dy) <= tol + 1.01 * out * np.abs(dy) + tiny)
    tol = eg.T @ np.abs(y) + (n + 64) * U * (np.abs(g).T @ np.abs(y))
    assert np.all(np.abs(got_dw - dw) <= tol + 1.01 * out * np.abs(dw) + tiny)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("gloss", [False, True])
def test_loss_scale_is_a_factor(dev, name, gloss):
    """A power of two changes no bit but where a result is subnormal without it."""
    n, d, k = 300, 40, 500
    x, w, lab = _inputs(n, d, k, 3)
    up = np.random.default_rng(1).random(n).astype(np.float32) + 0.5 if gloss else None
    plain = Run(dev, x, w, lab, name, gloss=up)
    px, pw, lb = R.Padded(dev, x, name), R.Padded(dev, w, name), dev.upload_u32(lab)
    lse = dev.upload_f32(plain.lse)
    dx, dw = (R.Padded(dev, np.zeros(s), name) for s in ((n, d), (k, d)))
    dev.cross_entropy_grad(px.buf, n, d, pw.buf, k, lb, lse, dx.buf, dw.buf, loss_scale=64.0,
                           gloss=None if up is None else dev.upload_f32(up))
    # (The least normal number itself may be what a subnormal one was rounded to.)
    least = 0.0 if name != "f16" else 2.0 ** -14
    for got, want in ((dx.read(), plain.dx), (dw.read(), plain.dw)):
        normal = (np.abs(want) > least) | (least == 0.0)
        assert np.array_equal(got[normal], 64.0 * want[normal])
        assert np.all(np.abs(got - 64.0 * want)[~normal] <= 64.0 * 2.0 ** -25)


def test_a_loss_scale_that_is_not_finite_is_refused(dev):
    from emeans_amd import EmeansHipInvalid, F32, U32
    z = lambda n: dev.zeros(n, F32)  # noqa: E731
    with pytest.raises(EmeansHipInvalid):
        dev.cross_entropy_grad(z(6), 2, 3, z(12), 4, dev.zeros(2, U32), z(2), z(6), z(12),
                               loss_scale=float("inf"))
    with pytest.raises(EmeansHipInvalid):
        dev.cross_entropy_grad(z(6), 2, 3, z(12), 4, dev.zeros(2, U32), z(2), z(6), z(12),
                               scale=1e30, loss_scale=1e30)
