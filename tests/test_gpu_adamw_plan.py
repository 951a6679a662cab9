"""An AdamW plan and the context that it was made with, in either order of their ends."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _plan(dev):
    from emeans_amd import F32, AdamTensor, AdamW
    p, g = dev.upload_f32(np.ones(1000)), dev.upload_f32(np.ones(1000))
    return p, AdamW(dev, [AdamTensor(p, g, dev.zeros(1000, F32), dev.zeros(1000, F32))])


def test_a_plan_whose_device_is_closed():
    from emeans_amd import EmeansHipInvalid, HipDevice
    dev = HipDevice()
    _, plan = _plan(dev)
    _, other = _plan(dev)
    plan.step(lr=1e-3, step=1)
    other.close()
    dev.close()
    with pytest.raises(EmeansHipInvalid, match="context"):
        plan.step(lr=1e-3, step=2)
    plan.close()
    with pytest.raises(EmeansHipInvalid):
        plan.step(lr=1e-3, step=2)


def test_a_plan_of_another_device_goes_on():
    from emeans_amd import HipDevice
    a, b = HipDevice(), HipDevice()
    _, gone = _plan(a)
    p, plan = _plan(b)
    plan.step(lr=1e-2, step=1)
    a.close()
    plan.step(lr=1e-2, step=2)
    assert np.abs(b.read_f32(p) - 0.98).max() < 1e-5
    gone.close()
    plan.close()
    b.close()
