"""Gradient norms at the end of f32's range."""

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


@pytest.mark.parametrize("mag,scale", [(3e38, 1.0), (1e30, 1e10), (-2e38, 1.0)])
@pytest.mark.parametrize("most", [1.0, 3e38, float("inf")])
def test_a_norm_beyond_f32_changes_nothing(dev, mag, scale, most):
    """Finite in f64, but not in f32: as any norm that is not finite."""
    from emeans_amd import F32, AdamTensor, AdamW, GradNorm
    x = np.full(1000, mag, np.float32)
    g, o, b = dev.upload_f32(x), dev.zeros(1000, F32), dev.zeros(2, F32)
    for plan in (GradNorm(dev, [g]), GradNorm(dev, [g], [o])):
        for call in (plan.norm, plan.clip):
            dev.write(b, 0, [7.0, 7.0])
            call(b, most, scale)
            got = dev.read(b)
            assert np.isposinf(got[0]) and np.isnan(got[1])
    assert dev.read(g).tobytes() == x.tobytes() and dev.read(o).tobytes() == x.tobytes()
    p, m, v = dev.upload_f32(np.ones(1000)), dev.zeros(1000, F32), dev.zeros(1000, F32)
    AdamW(dev, [AdamTensor(p, g, m, v)]).step(1e-2, 1, clip=b)
    assert (dev.read(p) == 1).all() and not dev.read(m).any() and not dev.read(v).any()


def test_the_largest_norm_of_f32_is_clipped(dev):
    from emeans_amd import F32, GradNorm
    x = np.full(3, 1.9e38, np.float32)
    g, b = dev.upload_f32(x), dev.zeros(2, F32)
    GradNorm(dev, [g]).clip(b, 1e10)
    norm = float(x[0]) * np.sqrt(3)
    got = dev.read(b)
    assert abs(got[0] - norm) <= 2 * R.U32 * norm and abs(got[1] * norm / 1e10 - 1) <= 2 * R.U32
    assert np.abs(dev.read(g) * np.sqrt(3) / 1e10 - 1).max() <= 4 * R.U32
