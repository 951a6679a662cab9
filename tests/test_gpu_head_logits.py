"""ClusterHead answers from f32 logits, whatever kind of rows it has."""

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


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [3, 500])
def test_answers_have_the_logits_of_f32(dev, n, norm, name):
    """Classes whose logits are some hundreds: log probabilities are off by what f32 sums of exact
    products are, where 16 bits are up to 0.25 (f16) or 2 (bf16) apart."""
    from emeans_amd.head import ClusterHead
    d, k, top = 200, 333, 5
    r = np.random.default_rng(n)
    x = r.standard_normal((n, d)).astype(np.float32)
    head = ClusterHead(d, k, kind=R.kind(name), centroids=20 * r.standard_normal((k, d)),
                       dev=dev, norm=norm)
    xb, lb = head.rows(x), head.labels(r.integers(0, k, n))
    got = head.answer(xb, n, top, lb)
    q, s = A.CodeBuf(dev, n, d), R.Padded(dev, np.zeros((n, A.blocks(d))), "f32")
    if norm == "rms":
        dev.rms_norm(xb, n, d, head.norm_weight, q.buf, scales=s.buf, eps=head.EPS)
    else:
        y = dev.zeros(n * d, R.kind(name))
        dev.layer_norm(xb, n, d, head.norm_weight, head.norm_bias, y, eps=head.EPS)
        dev.quantize(y, n, d, q.buf, s.buf)
    wq, ws = A.quantize(dev.read_f32(head.w).reshape(k, d), 128)
    a = R.f8_decode(q.read()) * A.spread(s.read(), 1, n, d)
    b = R.f8_decode(wq) * A.spread(ws, 128, k, d)
    z, mag = a @ b.T, np.abs(a) @ np.abs(b).T
    assert np.abs(z).max() > 500
    ref = A.LogProbs(z)
    # A logit: 128 roundings of a block's partial sums, a few of the scales and blocks, and its
    # own. It moves and lse moves; log_probs itself: differences, sums and their logarithm.
    tol = 2 * (140 * U * mag).max(1) + 4 * U * np.abs(z).max(1) + (k / 64 + 96) * U
    lp = lambda ids: np.take_along_axis(ref.lp, ids.astype(int), 1)  # noqa: E731
    assert np.all(np.abs(got.given - lp(dev.read(lb)[:, None])[:, 0]) <= tol + 2 * U * np.abs(got.given))
    assert np.all(np.abs(got.logp - lp(got.ids)) <= tol[:, None] + 2 * U * np.abs(got.logp))
    left = ref.lp.copy()
    np.put_along_axis(left, got.ids.astype(int), -np.inf, 1)
    assert np.all(left.max(1) <= got.logp[:, -1] + 2 * tol)
    assert np.all(np.diff(got.logp, axis=1) <= 0)
