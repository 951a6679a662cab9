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


LOW = {"f32": float(np.finfo(np.float32).min), "f16": -65504.0, "bf16": -(2.0 - 2.0 ** -7) * 2.0 ** 127}


def _large_rows(n, k, name):
    """Rows masked by the lowest value, wholly or but for one; two alike far above the others;
    one among masked ones; all far below zero, two of them less so; large ones of both signs."""
    low, big, far = LOW[name], *((60000.0, 60000.0) if name == "f16" else (1e10, 1e30))
    z = np.zeros((n, k))
    z[0] = low
    z[1] = low
    z[1, 7] = 5.0
    z[2, [3, k - 2]] = big
    z[3] = low
    z[3, k // 2] = far
    z[4] = -far
    z[4, [1, k - 1]] = -far / 2
    z[5] = np.random.default_rng(k).choice([-far, far, far / 4], k)
    return z, np.array([7, 7, 3, k // 2, 1, 0] + [0] * (n - 6))


class Exact:
    """The same in 64 bits from differences (beside 1e38 these hold no logarithm of a sum)."""

    def __init__(self, z, scale):
        with np.errstate(invalid="ignore"):
            m = z.max(1)
            self.none = np.isneginf(m)
            self.d = np.where(self.none[:, None], -np.inf, scale * (z - m[:, None]))
        s = np.where(self.none, 1.0, np.exp(self.d).sum(1))
        self.lp = self.d - np.log(s)[:, None]
        self.lse = scale * m + np.log(s)
        self.p = np.exp(self.lp)
        self.h = -np.where(self.p > 0, self.p * np.where(self.p > 0, self.lp, 0), 0.0).sum(1)
        self.order = np.argsort(-z, axis=1, kind="stable")

    def top(self, m):
        lp = np.take_along_axis(self.lp, self.order[:, :m], 1)
        return np.where(np.isneginf(lp), A.NONE, self.order[:, :m]), lp


@pytest.mark.parametrize("n,k", SHAPES)
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [0.7, 0.3, 1.3, 1e-30])
def test_large_logits_and_a_scale_whose_products_are_not_exact(dev, n, k, name, scale):
    """d = scale (z - m) is 0 for the largest, by each of k classes that are as large; a logit that
    the scale makes -infinite is none."""
    scale = float(np.float32(scale))
    z, tokens = _large_rows(n, k, name)
    (lp, lse, h, ids, tops), bufs = _call(dev, z, tokens, name, scale, 5)
    v = bufs[0].value
    with np.errstate(over="ignore"):
        v = np.where(np.isneginf((v * scale).astype(np.float32)), -np.inf, v)
    ref = Exact(v, scale)
    # Sums of equal terms, or of one and what rounds to nothing beside it (1e-30: of k alike).
    s = 4 * (k / 64 + 96) * U * (1 + np.log(k))

    def near(a, b):
        with np.errstate(invalid="ignore"):
            return (a == b) | (np.abs(a - b) <= s + 4 * U * np.abs(b))
    wi, wl = ref.top(5)
    assert near(lse, ref.lse).all() and near(h, ref.h).all()
    assert near(lp, ref.lp[np.arange(n), tokens]).all()
    assert np.array_equal(ids, wi) and near(tops, wl).all()


@pytest.mark.parametrize("n,k", SHAPES)
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [0.7, 0.3, 1.0])
def test_gradients_of_large_logits(dev, n, k, name, scale):
    """Rows that count nothing get zeros whatever their logits, and all of them finite values; a
    class that is alone has p = 1, and its row no gradient."""
    scale = float(np.float32(scale))
    z, tokens = _large_rows(n, k, name)
    _, bufs = _call(dev, z, tokens, name, scale, 0)
    zero, one = np.zeros(n), np.random.default_rng(3).standard_normal(n)
    assert (_grad(dev, bufs, scale, zero, zero) == 0).all()
    g = _grad(dev, bufs, scale, one, one)
    assert np.isfinite(g).all()
    assert (g[[1, 3]] == 0).all()
    assert g[6:].any() or n == 6


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [1.0, 0.7])
@pytest.mark.parametrize("size", [20.0, 3000.0, 60000.0])
def test_how_far_a_gradient_of_large_logits_is_off(dev, name, scale, size):
    """Two classes alike far above the others: p is a half, off by a factor within exp(2^-23 |lse|)
    and the roundings of lse's own logarithm and of the result."""
    scale = float(np.float32(scale))
    n, k = 3, 1000
    z = np.full((n, k), -size)
    z[:, [1, 998]] = size
    (lp, lse, h, _, _), bufs = _call(dev, z, np.ones(n), name, scale, 0)
    assert np.abs(lp + np.log(2)).max() <= 200 * U and np.abs(h - np.log(2)).max() <= 200 * U
    g = _grad(dev, bufs, scale, np.ones(n), np.zeros(n))
    off = np.expm1(2.0 ** -23 * scale * size) + 200 * U
    want = np.array([0.5, -0.5]) * scale
    assert np.all(np.abs(g[:, [1, 998]] - want) <= scale * 0.5 * off + R.UNIT[name] * scale)
    assert (np.delete(g, [1, 998], 1) == 0).all() or size == 20.0


@pytest.mark.parametrize("n,k", SHAPES)
@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_classes_whose_log_probability_is_beyond_f32(dev, n, k, name):
    """Their logits are finite: they are among the likeliest, in their order, with -infinity."""
    z = np.full((n, k), -np.inf)
    z[:, [2, 5, k - 1]] = -3e38, -2e38, 3e38
    (lp, lse, h, ids, tops), _ = _call(dev, z, np.full(n, 2), name, 1.0, 4)
    assert np.isneginf(lp).all() and (h == 0).all() and np.isfinite(lse).all()
    assert (ids == [k - 1, 5, 2, A.NONE]).all()
    assert (tops[:, 0] == 0).all() and np.isneginf(tops[:, 1:]).all()
