"""8-bit AdamW over thousands of steps against 32-bit states on the same gradients: with a
seed the second moment follows gradients that change their size inside a block."""

import numpy as np
import pytest

from tests import learn_ref as R

pytestmark = pytest.mark.gpu
STEPS, CHANGE = 4000, 1000


@pytest.fixture(scope="module")
def dev():
    from emeans_amd import HipDevice
    d = HipDevice()
    yield d
    d.close()


class Pair:
    """One tensor with 32-bit and one with 8-bit states, one gradient buffer."""

    def __init__(self, dev, n, seed=3, gkind=None):
        from emeans_amd import F32, F8, AdamTensor, AdamW
        self.dev, self.n = dev, n
        self.grad = dev.zeros(n, F32)
        blocks = -(-n // AdamW.BLOCK)
        self.p = [dev.zeros(n, F32) for _ in range(2)]
        self.m, self.v = ([dev.zeros(n, k) for k in (F32, F8)] for _ in range(2))
        self.ms, self.vs = (dev.zeros(blocks, F32) for _ in range(2))
        self.plans = [AdamW(dev, [AdamTensor(self.p[0], self.grad, self.m[0], self.v[0])]),
                      AdamW(dev, [AdamTensor(self.p[1], self.grad, self.m[1], self.v[1], self.ms,
                                             self.vs)], seed=seed)]

    def step(self, g, step, lr=1e-3, **hyper):
        self.dev.write(self.grad, 0, g)
        for plan in self.plans:
            plan.step(lr=lr, step=step, **hyper)

    def roots(self):
        scale = np.repeat(self.dev.read(self.vs).astype(float), 256)[:self.n]
        return (np.sqrt(self.dev.read(self.v[0]).astype(float)),
                R.f8_decode(self.dev.read(self.v[1])) * scale)


@pytest.mark.parametrize("factor", [1.0, 0.1, 4.0])
@pytest.mark.parametrize("n", [2048, 5001])
def test_the_second_moment_follows(dev, n, factor):
    """Every other element's gradients change by the factor after a while. A root that is
    rounded at random wanders: a step adds (1 - beta2) / 2 |g^2 / v - 1| of a code's step
    times that step (9 % of it), twice (the block's scale moves as well), and the average
    forgets (1 - beta2) of it: a variance of about (0.0005 + 0.0005) 0.09 / 0.002, a fifth of
    its size. So the mean over a thousand elements is within a tenth, and nine in ten
    are within half of it."""
    r = np.random.default_rng(n)
    size = np.exp(r.standard_normal(n)) * 1e-3
    pair = Pair(dev, n)
    for t in range(1, STEPS + 1):
        g = (r.standard_normal(n) * size).astype(np.float32)
        if t > CHANGE:
            g[::2] *= np.float32(factor)
        pair.step(g, t)
    want, got = pair.roots()
    for half in (slice(0, None, 2), slice(1, None, 2)):
        ratio = got[half] / want[half]
        assert 0.9 < ratio.mean() < 1.1
        assert np.mean((ratio > 0.5) & (ratio < 1.5)) > 0.9
    # The steps taken, by their sizes: a random walk of 4,000 steps of both, which agree
    # but for the roots' and m's own errors.
    moved = [np.sqrt((dev.read(p).astype(float) ** 2).mean()) for p in pair.p]
    assert 0.8 < moved[1] / moved[0] < 1.25


def test_a_constant_gradient_is_followed_down_to_its_size(dev):
    """m and the root of a gradient of one size settle at it whatever they were before."""
    n = 1024
    pair = Pair(dev, n)
    for t in range(1, 501):
        pair.step(np.full(n, 1.0 if t < 20 else 1e-2, np.float32), t, beta2=0.98)
    want, got = pair.roots()
    assert np.all(np.abs(want - 1e-2) < 1e-3)
    assert abs(got.mean() / want.mean() - 1) < 0.1


@pytest.mark.parametrize("n", [1, 255, 1024, 5001])
def test_one_step_takes_the_codes_around_a_value(dev, n):
    """Each code is one of the two around value / scale, on average (over seeds) the value;
    the parameters and scales are those of the nearest rounding."""
    from emeans_amd import F32, F8, AdamTensor, AdamW
    r = np.random.default_rng(n)
    g = (r.standard_normal(n) * np.exp(2 * r.standard_normal(n))).astype(np.float32)
    grad, blocks, seeds = dev.upload_f32(g), -(-n // 256), 64
    table = np.concatenate([R.F8[:127], [np.inf]])

    def run(seed):
        p, m, v = dev.zeros(n, F32), dev.zeros(n, F8), dev.zeros(n, F8)
        ms, vs = dev.zeros(blocks, F32), dev.zeros(blocks, F32)
        AdamW(dev, [AdamTensor(p, grad, m, v, ms, vs)], seed=seed).step(lr=1e-3, step=1)
        return [dev.read(b) for b in (p, m, v, ms, vs)]

    near, runs = run(None), [run(s) for s in range(seeds)]
    again = run(5)
    assert all(np.array_equal(a, b) for a, b in zip(again, runs[5]))
    assert n < 64 or any(not np.array_equal(runs[0][1], a[1]) for a in runs[1:])
    for want, at, sc in ((0.1 * g.astype(float), 1, 3), (np.sqrt(1e-3) * np.abs(g.astype(float)), 2, 4)):
        total = np.zeros(n)
        for a in runs:
            assert np.array_equal(a[0], near[0]) and np.array_equal(a[sc], near[sc])
            scale = np.repeat(a[sc].astype(float), 256)[:n]
            q = np.abs(want) / scale
            got = np.abs(R.f8_decode(a[at]))
            i = np.searchsorted(table, q * (1 - 1e-6), side="right") - 1
            j = np.searchsorted(table, q * (1 + 1e-6), side="left")
            least = 2.0 ** -9 if at == 2 else 0.0
            assert np.all((got >= table[i]) & (got <= np.maximum(table[np.minimum(j, 126)], least)))
            assert np.all((R.f8_decode(a[at]) >= 0) | (want < 0))
            total += got
        # 64 draws of a step of at most q / 8 (or 2^-9): five deviations of their mean.
        mean, spread = total / seeds, np.maximum(q / 8, 2.0 ** -9) / 2 / np.sqrt(seeds)
        assert np.all((np.abs(mean - q) <= 5 * spread + 1e-6 * q) | (q < least))


def test_values_that_are_not_finite(dev):
    from emeans_amd import F32, F8, AdamTensor, AdamW
    g = np.ones(512, np.float32)
    g[3], g[300] = np.nan, np.inf
    p, m, v = dev.zeros(512, F32), dev.zeros(512, F8), dev.zeros(512, F8)
    ms, vs = dev.zeros(2, F32), dev.zeros(2, F32)
    AdamW(dev, [AdamTensor(p, dev.upload_f32(g), m, v, ms, vs)], seed=1).step(lr=1e-3, step=1)
    for b in (m, v):
        got = R.f8_decode(dev.read(b))
        bad = np.isnan(got)
        assert bad[3] and bad[300] and bad.sum() == 2
        assert np.all(got[~bad] == 448.0)
