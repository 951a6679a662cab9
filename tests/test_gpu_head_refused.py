"""What ClusterHead refuses leaves it as it was."""

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
