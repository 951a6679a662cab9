"""The learning operators run together: ClusterHead's steps against the same training in
64 bits, in every kind and both state widths, on labels from a clustering."""

import numpy as np
import pytest

from tests import learn_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from emeans_amd import HipDevice
    d = HipDevice()
    yield d
    d.close()


@pytest.fixture(scope="module")
def clustered(dev):
    from emeans_amd import Config, Emeans, synth
    x, _ = synth.blobs_spherical(3000, 48, 20, 0.1, seed=3)
    model = Emeans(Config(d=48, k=20, spherical=True, seed=3), dev)
    labels = model.train(x).labels.copy()
    labels[::17] = -1
    return np.asarray(x, np.float32).reshape(-1, 48), labels, model.centroids().reshape(20, 48)


class Reference:
    """The same training in 64 bits."""

    def __init__(self, w, scale=1.0, decay=0.01):
        d = w.shape[1]
        self.p = [w.astype(float).copy(), np.ones(d), np.zeros(d)]
        self.m = [np.zeros_like(a) for a in self.p]
        self.v = [np.zeros_like(a) for a in self.p]
        self.scale, self.decay, self.t = scale, [decay, 0.0, 0.0], 0

    def step(self, x, lab, lr):
        self.t += 1
        w, g, b = self.p
        y, _, rstd, h = R.layer_norm(x, g, b, 1e-5)
        loss, _, p, _ = R.cross_entropy(y, w, lab, self.scale)
        has = lab != 0xFFFFFFFF
        up = np.where(has, 1.0 / max(1, has.sum()), 0.0)
        dy, dw, _ = R.cross_entropy_grad(y, w, lab, self.scale, p, up)
        _, dg, db = R.layer_norm_grad(dy, h, rstd, g)
        for i, grad in enumerate((dw, dg, db)):
            self.m[i] = 0.9 * self.m[i] + 0.1 * grad
            self.v[i] = 0.999 * self.v[i] + 0.001 * grad * grad
            by = (self.m[i] / (1 - 0.9 ** self.t)) / (np.sqrt(self.v[i] / (1 - 0.999 ** self.t)) + 1e-8)
            self.p[i] = self.p[i] * (1 - lr * self.decay[i]) - lr * by
        return loss


@pytest.mark.parametrize("name,bits", [("f32", 32), ("f32", 8), ("bf16", 32), ("bf16", 8), ("f16", 8)])
def test_steps_follow_the_64_bit_training(dev, clustered, name, bits):
    """Eight steps on one batch. A step moves a weight by at most about lr whatever the
    gradient's size, so a gradient's error shows where it changes sign: an element whose
    gradient is within its error of zero. f32: 1e-3 of lr on average; 16 bits and
    8-bit states: a few hundredths of the distance moved."""
    from emeans_amd.head import ClusterHead
    x, labels, cent = clustered
    lr = 1e-3
    head = ClusterHead(48, 20, kind=R.kind(name), state_bits=bits, centroids=cent, dev=dev)
    ref = Reference(cent)
    xb, lb = head.rows(x), head.labels(labels)
    x64 = R.decode(R.encode(x, name), name)
    lab = np.where(labels < 0, 0xFFFFFFFF, labels).astype(np.uint32)
    first = None
    for _ in range(8):
        loss = dev.read_f32(head.step(xb, lb, len(x), lr))[:len(x)]
        want = ref.step(x64, lab, lr)
        # Rows normalized to 16 bits, classes in 16 bits: logits of up to 8 within 2^-8 of that.
        tol = 1e-3 if name == "f32" else 8 * 4 * R.UNIT[name]
        tol += 0.0 if bits == 32 else 8 * lr
        assert np.abs(loss - want).max() <= tol
        assert not loss[labels < 0].any()
        first = want.sum() if first is None else first
    assert want.sum() < first  # it learns
    far = 0.002 if (name, bits) == ("f32", 32) else 0.1
    for got, p, start in ((head.w, ref.p[0], cent), (head.norm_weight, ref.p[1], np.ones(48)),
                          (head.norm_bias, ref.p[2], np.zeros(48))):
        off = np.abs(dev.read_f32(got).astype(float).reshape(p.shape) - p)
        assert off.mean() <= far * np.abs(p - start).mean()


def test_fit_from_host_rows(dev, clustered):
    from emeans_amd import BF16
    from emeans_amd.head import ClusterHead
    x, labels, _ = clustered
    head = ClusterHead(48, 20, kind=BF16, state_bits=8, dev=dev, seed=5)
    losses = head.fit(x, labels, epochs=6, batch=700, lr=1e-2)
    assert losses[0] < 4.0 and losses[-1] < 0.5 * losses[0] and np.isfinite(losses).all()
    again = ClusterHead(48, 20, kind=BF16, state_bits=8, dev=dev, seed=5)
    assert again.fit(x, labels, epochs=6, batch=700, lr=1e-2) == losses  # the same bits
    held = again.loss(again.rows(x[:100]), again.labels(labels[:100]), 100)
    assert held.shape == (100,) and (held >= 0).all()


def test_refusals(dev):
    from emeans_amd import F8
    from emeans_amd.head import ClusterHead
    for bad in (dict(d=0), dict(k=0), dict(kind=F8), dict(state_bits=16),
                dict(centroids=np.zeros(7))):
        with pytest.raises(ValueError):
            ClusterHead(**{**dict(d=8, k=4, dev=dev), **bad})
    head = ClusterHead(8, 4, dev=dev)
    with pytest.raises(ValueError):
        head.rows(np.zeros(9))
    with pytest.raises(ValueError):
        head.fit(np.zeros((5, 8)), np.zeros(4, np.int32))
    with pytest.raises(ValueError):
        head.fit(np.zeros((5, 8)), np.zeros(5, np.int32), batch=0)
