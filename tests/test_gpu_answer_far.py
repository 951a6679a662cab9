"""The answering and tuning operators on matrices whose elements 32 bits do not number: rows far
apart, and many of them, against the same calls on the rows that matter alone. (A row's result
follows from its own elements, so the two are equal to the last bit where the same sums are
made.)"""

import numpy as np
import pytest

from tests import answer_ref as A

pytestmark = pytest.mark.gpu
FAR = 1 << 31  # a row's stride: the third begins at element 2^32


@pytest.fixture(scope="module")
def dev():
    from emeans_amd import HipDevice
    d = HipDevice()
    yield d
    d.close()


class Rows:
    """Three rows FAR apart, and a buffer of them side by side."""

    def __init__(self, dev, d, kind, a=None):
        self.dev, self.d = dev, d
        self.far, self.near = dev.zeros(2 * FAR + (-(-d // 16) * 16), kind), dev.zeros(3 * (-(-d // 16) * 16), kind)
        if a is not None:
            for i in range(3):
                dev.write(self.far, i * FAR, a[i])
                dev.write(self.near, i * d, a[i])

    def pairs(self, near_ld):
        for i in range(3):
            f = self.dev.read(self.far, (i * FAR, i * FAR + self.d))
            n = self.dev.read(self.near, (i * near_ld, i * near_ld + self.d))
            assert n.any()
            yield f, n

    def equal(self, near_ld):
        return all(f.tobytes() == n.tobytes() for f, n in self.pairs(near_ld))


SUMS = 32 * 2.0 ** -24


def close(a, b, rel):
    """Off by at most rel of the larger (f16's least step apart)."""
    a, b = a.astype(float), b.astype(float)
    return np.all(np.abs(a - b) <= rel * np.maximum(np.abs(a), np.abs(b)) + 2.0 ** -24)


def test_rms_norm_and_its_gradient(dev):
    from emeans_amd import F16, F32
    d = 100
    r = np.random.default_rng(1)
    x, dy = (Rows(dev, d, F16, r.standard_normal((3, d))) for _ in range(2))
    y, dx = Rows(dev, d, F16), Rows(dev, d, F16)
    rstd, dw = [dev.zeros(3, F32) for _ in range(2)], [dev.zeros(d, F32) for _ in range(2)]
    dev.rms_norm(x.far, 3, d, None, y.far, rstd=rstd[0], ldx=FAR, ldy=FAR)
    dev.rms_norm(x.near, 3, d, None, y.near, rstd=rstd[1])
    assert y.equal(d) and dev.read(rstd[0]).tobytes() == dev.read(rstd[1]).tobytes()
    dev.rms_norm_grad(dy.far, x.far, 3, d, None, rstd[0], dx.far, dw[0], lddy=FAR, ldh=FAR, lddx=FAR)
    dev.rms_norm_grad(dy.near, x.near, 3, d, None, rstd[1], dx.near, dw[1])
    assert dx.equal(d) and dev.read(dw[0]).tobytes() == dev.read(dw[1]).tobytes()


def test_codes_and_their_product(dev):
    from emeans_amd import F8, F16, F32
    d, k = 112, 70
    r = np.random.default_rng(2)
    x = Rows(dev, d, F16, r.standard_normal((3, d)))
    q, s = Rows(dev, d, F8), [dev.zeros(3, F32) for _ in range(2)]
    dev.quantize(x.far, 3, d, q.far, s[0], ldx=FAR, ldq=FAR)
    dev.quantize(x.near, 3, d, q.near, s[1])
    assert q.equal(d) and dev.read(s[0]).tobytes() == dev.read(s[1]).tobytes()
    w, w8, ws = dev.upload_f32(r.standard_normal((k, d))), dev.zeros(k * d, F8), dev.zeros(1, F32)
    dev.quantize(w, k, d, w8, ws, tile_rows=dev.CODE_BLOCK)
    y = Rows(dev, k, F16)
    dev.product8(q.far, s[0], 3, d, w8, ws, k, y.far, ldx=FAR, ldy=FAR)
    dev.product8(q.near, s[1], 3, d, w8, ws, k, y.near)
    assert y.equal(k)
    # The classes far apart: three of them, and as many columns.
    out = [dev.zeros(9, F32) for _ in range(2)]
    dev.product8(q.near, s[1], 3, d, q.far, s[0], 3, out[0], ldw=FAR)
    dev.product8(q.near, s[1], 3, d, q.near, s[1], 3, out[1])
    assert dev.read(out[0]).tobytes() == dev.read(out[1]).tobytes()


def test_log_probs_and_their_gradient(dev):
    from emeans_amd import F16, F32, U32
    k, top = 333, 3
    r = np.random.default_rng(3)
    z, dz = Rows(dev, k, F16, 2 * r.standard_normal((3, k))), Rows(dev, k, F16)
    t, g = dev.upload_u32(np.array([5, 332, 0], np.uint32)), dev.upload_f32(np.array([1.0, -2, 3]))
    out = []
    for m, ld in ((z.far, FAR), (z.near, 0)):
        lp, lse, h, tops = (dev.zeros(c, F32) for c in (3, 3, 3, 3 * top))
        ids = dev.zeros(3 * top, U32)
        dev.log_probs(m, 3, k, t, lp, lse, entropy=h, top=top, top_ids=ids, top_logp=tops, ldz=ld)
        out.append((lp, lse, h, ids, tops))
    for a, b in zip(*out):  # (log probabilities are up to 10 and more)
        assert close(dev.read(a), dev.read(b), SUMS)
    lse, h = out[0][1], out[0][2]
    dev.log_probs_grad(z.far, 3, k, t, lse, dz.far, entropy=h, glogp=g, gentropy=g, ldz=FAR, lddz=FAR)
    dev.log_probs_grad(z.near, 3, k, t, lse, dz.near, entropy=h, glogp=g, gentropy=g)
    assert all(close(f, m, 2.0 ** -10) for f, m in dz.pairs(k))


def test_many_rows(dev):
    """131,075 rows by 32,769 classes, 2^32 logits and more: a product, its log probabilities and
    their gradient; the last rows against a call on them alone."""
    from emeans_amd import F8, F16, F32, U32
    n, k, d, top, last = (1 << 17) + 3, (1 << 15) + 1, 16, 2, 4
    r = np.random.default_rng(4)
    q, s = dev.zeros(n * d, F8), dev.zeros(n, F32)
    codes, _ = A.quantize(r.standard_normal((n, d)), 1)
    dev.write(q, 0, codes.reshape(-1))
    dev.write(s, 0, r.uniform(0.001, 0.002, n))
    w8, ws = dev.zeros(k * d, F8), dev.zeros(dev.code_blocks(k), F32)
    dev.quantize(dev.upload_f32(r.standard_normal((k, d))), k, d, w8, ws, tile_rows=dev.CODE_BLOCK)
    y = dev.zeros(n * k, F16)
    dev.product8(q, s, n, d, w8, ws, k, y)
    at = n - last
    part = lambda b, size, c: dev.wrap(b.ptr + at * c * size, last * c, b.kind)  # noqa: E731
    few = dev.zeros(last * k, F16)
    dev.product8(part(q, 1, d), part(s, 4, 1), last, d, w8, ws, k, few)
    got, want = (dev.read(b, rng).astype(float) for b, rng in ((y, (at * k, n * k)), (few, None)))
    # One block of two eights of products: either way off by 7 2^-13 of the largest of each eight
    # and one rounding.
    largest = (448 * 0.002) * (448 * dev.read(ws).max())
    tol = 2 * (2 * 7 * 2.0 ** -13 * largest + 2.0 ** -11 * np.abs(want).max())
    assert np.abs(want).max() > 100 * tol and np.abs(got - want).max() <= tol
    dev.write(few, 0, got.astype(np.float16))
    t = dev.upload_u32(r.integers(0, k, n).astype(np.uint32))
    lp, lse, h, tops = (dev.zeros(c, F32) for c in (n, n, n, n * top))
    ids = dev.zeros(n * top, U32)
    dev.log_probs(y, n, k, t, lp, lse, entropy=h, top=top, top_ids=ids, top_logp=tops)
    ref = A.LogProbs(got.reshape(last, k))
    assert np.array_equal(dev.read(ids, (at * top, n * top)).reshape(last, top), ref.top(top)[0])
    assert close(dev.read(lse, (at, n)), ref.lse, 2 * SUMS)
    g = dev.upload_f32(r.standard_normal(n))
    dev.log_probs_grad(y, n, k, t, lse, y, entropy=h, glogp=g, gentropy=g)  # in its place
    dz = dev.zeros(last * k, F16)
    dev.log_probs_grad(few, last, k, part(t, 4, 1), part(lse, 4, 1), dz, entropy=part(h, 4, 1),
                       glogp=part(g, 4, 1), gentropy=part(g, 4, 1))
    assert close(dev.read(y, (at * k, n * k)), dev.read(dz), 2.0 ** -10)


def test_a_long_gradient(dev):
    """2^32 + 5 elements: the last ones count, and are scaled."""
    from emeans_amd import F16, F32, GradNorm
    n = (1 << 32) + 5
    g, out = dev.zeros(n, F16), dev.zeros(2, F32)
    dev.write(g, 0, [3.0])
    dev.write(g, n - 2, [4.0, 12.0])
    plan = GradNorm(dev, [g])
    plan.clip(out, 6.5)
    assert dev.read(out).tolist() == [13.0, 0.5]
    assert dev.read(g, (0, 2)).tolist() == [1.5, 0.0]
    assert dev.read(g, (n - 4, n)).tolist() == [0.0, 0.0, 2.0, 6.0]
