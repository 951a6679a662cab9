"""What ClusterHead refuses, which leaves it as it was, and what it takes."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from emeans_amd import HipDevice
    d = HipDevice()
    yield d
    d.close()


def test_a_refused_step_does_not_count(dev):
    from emeans_amd import EmeansHipInvalid
    from emeans_amd.head import ClusterHead
    r = np.random.default_rng(2)
    x, lab = r.standard_normal((20, 8)), r.integers(0, 4, 20)

    def run(refuse):
        head = ClusterHead(8, 4, dev=dev, seed=1)
        xb, lb = head.rows(x), head.labels(lab)
        for _ in range(2):
            if refuse:
                with pytest.raises(EmeansHipInvalid):
                    head.step(xb, lb, 21, 1e-2)
                with pytest.raises(EmeansHipInvalid):
                    head.step(xb, lb, 20, float("nan"))
            head.step(xb, lb, 20, 1e-2)
        assert head.steps == 2
        return dev.read_f32(head.w)

    assert np.array_equal(run(True), run(False))


def test_labels_of_more_than_32_bits(dev):
    from emeans_amd import NONE
    from emeans_amd.head import ClusterHead
    head = ClusterHead(8, 4, dev=dev)
    with pytest.raises(ValueError):
        head.labels(np.array([1, (1 << 32) + 1]))
    for kind in (np.int8, np.int32, np.int64):
        assert list(dev.read_u32(head.labels(np.array([3, -1, -7], kind)))) == [3, NONE, NONE]
    assert list(dev.read_u32(head.labels(np.array([3, NONE], np.uint32)))) == [3, NONE]


def test_any_seed_that_numpy_takes(dev):
    from emeans_amd import BF16
    from emeans_amd.head import ClusterHead
    r = np.random.default_rng(2)
    x, lab = r.standard_normal((50, 8)), r.integers(0, 4, 50)

    def run(seed, **kw):
        head = ClusterHead(8, 4, kind=BF16, state_bits=8, dev=dev, seed=seed, **kw)
        return head.fit(x, lab, epochs=3, batch=20)

    for seed in (0, [1, 2], np.random.SeedSequence(5), 1 << 70):
        assert run(seed) == run(seed)
        assert run(seed, centroids=np.ones((4, 8))) == run(seed, centroids=np.ones((4, 8)))
    assert np.isfinite(run(None)).all()
