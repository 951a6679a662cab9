"""The global gradient norm and clipping against 64 bits, and the AdamW step that takes its
factor: tensors of every type and length at any address, in place and not, norms that are not
finite, graphs."""

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


LENGTHS = {"one": [1], "few": [3, 0, 7, 1000, 2048, 2049], "many": [17 * i % 301 for i in range(90)],
           "large": [3_000_001, 5, 2_500_000, 0, 16384]}


def _tensors(dev, lengths, seed, off):
    r = np.random.default_rng(seed)
    names = ["f32", "bf16", "f16"]
    return [R.Padded(dev, r.standard_normal((1, n)) * 10.0 ** r.integers(-2, 2), names[i % 3], 0,
                     (off * (i + 1)) % 9) for i, n in enumerate(lengths)]


def _views(dev, ts):
    return [dev.wrap(t.buf.ptr, t.d, t.buf.kind) for t in ts]


@pytest.mark.parametrize("which", list(LENGTHS))
@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("by", [0.3, 1.5])
def test_norm_and_clip(dev, which, off, by):
    from emeans_amd import F32, GradNorm
    ts = _tensors(dev, LENGTHS[which], len(which), off)
    outs = [R.Padded(dev, np.zeros((1, t.d)), t.name, 0, (t.off + 3) % 9, fill=7.0) for t in ts]
    scale = 0.25
    norm = scale * np.sqrt(sum((t.value ** 2).sum() for t in ts))
    most = np.float32(by * norm)
    b = dev.zeros(2, F32)
    apart = GradNorm(dev, _views(dev, ts), _views(dev, outs))
    apart.norm(b, scale=scale)
    got = dev.read(b)
    assert abs(got[0] - norm) <= 2 * U * norm and got[1] == 1
    apart.norm(b, most, scale)
    got = dev.read(b)
    want = min(1.0, float(most) / norm)
    assert abs(got[1] - want) <= 2 * U * want
    apart.clip(b, most, scale)
    assert np.array_equal(dev.read(b), got)
    here = GradNorm(dev, _views(dev, ts))
    here.clip(b, most, scale)
    assert np.array_equal(dev.read(b), got)
    for t, o in zip(ts, outs):
        f = np.float32(got[1])
        prod = (t.value.astype(np.float32) * f).astype(np.float32)  # (one rounding in f32)
        v = R.decode(R.encode(prod, t.name), t.name)
        assert np.array_equal(o.read(), v) and np.array_equal(t.read(), v)
    apart.close(), here.close()


def test_squares_beyond_f32(dev):
    from emeans_amd import F32, GradNorm
    for mag in (1e30, 1e-30):
        a = dev.upload_f32(np.full(5000, mag))
        b = dev.zeros(2, F32)
        GradNorm(dev, [a]).clip(b, mag)
        got = dev.read(b)
        want = float(np.float32(mag)) * np.sqrt(5000)
        assert abs(got[0] - want) <= 2 * U * want
        v = dev.read(a)
        assert abs(np.sqrt((v.astype(float) ** 2).sum()) - mag) <= 8 * U * mag


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_norm_that_is_not_finite_changes_nothing(dev, bad):
    from emeans_amd import F32, GradNorm
    x = np.ones(3000, np.float32)
    x[1234] = bad
    a, o, b = dev.upload_f32(x), dev.zeros(3000, F32), dev.zeros(2, F32)
    GradNorm(dev, [a]).clip(b, 0.5)
    got = dev.read(b)
    assert not np.isfinite(got[0]) and np.isnan(got[1])
    assert dev.read(a).tobytes() == x.tobytes()
    GradNorm(dev, [a], [o]).clip(b, 0.5)
    assert dev.read(o).tobytes() == x.tobytes()


def test_nothing_to_measure(dev):
    from emeans_amd import F32, GradNorm
    b = dev.upload_f32([5.0, 5.0])
    GradNorm(dev, []).clip(b, 1.0)
    assert dev.read(b).tolist() == [0.0, 1.0]
    b = dev.upload_f32([5.0, 5.0])
    GradNorm(dev, [dev.zeros(0, F32)]).norm(b, 0.0)
    assert dev.read(b).tolist() == [0.0, 1.0]
    a = dev.upload_f32(np.ones(10))
    GradNorm(dev, [a]).clip(b, 0.0)  # down to zero
    assert not dev.read(a).any()


@pytest.mark.parametrize("eight", [False, True])
def test_adamw_takes_the_factor(dev, eight):
    from emeans_amd import F32, F8, AdamTensor, AdamW, GradNorm
    n = 5000
    r = np.random.default_rng(1)
    p0, g0 = r.standard_normal(n).astype(np.float32), r.standard_normal(n).astype(np.float32)

    def make(g):
        p, gb = dev.upload_f32(p0), dev.upload_f32(g)
        if eight:
            m, v = dev.zeros(n, F8), dev.zeros(n, F8)
            ms, vs = dev.zeros(20, F32), dev.zeros(20, F32)
            t = AdamTensor(p, gb, m, v, ms, vs)
        else:
            m, v = dev.zeros(n, F32), dev.zeros(n, F32)
            t = AdamTensor(p, gb, m, v)
        return p, gb, m, v, AdamW(dev, [t])
    b = dev.zeros(2, F32)
    p, g, m, v, plan = make(g0)
    GradNorm(dev, [g]).norm(b, 3.0, 0.5)
    f = dev.read(b)[1]
    assert f < 0.2
    plan.step(1e-2, 1, grad_scale=0.5, clip=b)
    # What the step without it does with that grad_scale.
    p2, _, m2, v2, plan2 = make(g0)
    plan2.step(1e-2, 1, grad_scale=float(np.float32(0.5) * f))
    for x, y in ((p, p2), (m, m2), (v, v2)):
        assert dev.read(x).tobytes() == dev.read(y).tobytes()
    # A gradient that is not finite: nothing changes.
    g0 = g0.copy()
    g0[7] = np.inf
    p, g, m, v, plan = make(g0)
    GradNorm(dev, [g]).norm(b, 3.0)
    plan.step(1e-2, 1, clip=b)
    assert dev.read(p).tobytes() == p0.tobytes() and not dev.read(m).any() and not dev.read(v).any()


def test_refusals(dev):
    from emeans_amd import (F16, F32, U32, AdamTensor, AdamW, EmeansHipInvalid, GradNorm, HipDevice)
    a, o, b = dev.zeros(100, F32), dev.zeros(100, F32), dev.zeros(2, F32)

    def no(match, f):
        with pytest.raises(EmeansHipInvalid, match=match):
            f()
    no("grad must be", lambda: GradNorm(dev, [dev.zeros(3, U32)]))
    no("its output must be", lambda: GradNorm(dev, [a], [dev.zeros(99, F32)]))
    no("its output must be", lambda: GradNorm(dev, [a], [dev.zeros(100, F16)]))
    no("overlaps", lambda: GradNorm(dev, [a, dev.wrap(a.ptr, 10, F32)]))
    no("overlaps", lambda: GradNorm(dev, [a, o], [o, a]))
    no("overlaps", lambda: GradNorm(dev, [a], [dev.wrap(a.ptr + 4, 100, F32)]))
    no("overlaps", lambda: GradNorm(dev, [a, a], [o, o]))
    with pytest.raises(ValueError):
        GradNorm(dev, [a], [])
    GradNorm(dev, [a, a], [o, dev.zeros(100, F32)])  # a gradient may be read twice
    plan = GradNorm(dev, [a])
    no("max_norm", lambda: plan.norm(b, -1.0))
    no("max_norm", lambda: plan.norm(b, float("nan")))
    no("scale must be", lambda: plan.norm(b, 1.0, float("inf")))
    no("out must be", lambda: plan.norm(dev.zeros(2, U32)))
    no("out: the buffer's", lambda: plan.norm(dev.zeros(1, F32)))
    no("out overlaps", lambda: plan.norm(dev.wrap(a.ptr, 2, F32)))
    m, v = dev.zeros(100, F32), dev.zeros(100, F32)
    step = AdamW(dev, [AdamTensor(o, a, m, v)])
    no("clip must be", lambda: step.step(1e-3, 1, clip=dev.zeros(2, U32)))
    no("overlaps clip", lambda: step.step(1e-3, 1, clip=dev.wrap(m.ptr, 2, F32)))
    other = HipDevice()
    plan = GradNorm(other, [other.zeros(4, F32)])
    other.close()
    no("context is destroyed", lambda: plan.norm(b))


def test_a_captured_clip_replays(dev):
    from emeans_amd import F32, GradNorm
    r = np.random.default_rng(3)
    x = r.standard_normal(70_000).astype(np.float32)
    a, o, b = dev.upload_f32(x), dev.zeros(70_000, F32), dev.zeros(2, F32)
    plan = GradNorm(dev, [a], [o])
    dev.sync()
    g = A.Graph(dev, lambda: plan.clip(b, 10.0))
    for i in range(4):
        dev.write(a, 0, x * np.float32(0.01 * 10.0 ** i))
        dev.sync()
        g.replay()
        got = dev.read(o).tobytes(), dev.read(b).tobytes()
        plan.clip(b, 10.0)
        assert got == (dev.read(o).tobytes(), dev.read(b).tobytes())
    g.close()
