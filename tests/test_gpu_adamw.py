"""The AdamW step over lists of tensors against 64 bits, states in 32 and in 8
bits: lengths around the block and chunk sizes, every type of parameter and
gradient, addresses that suit no vector, and what it refuses."""

import numpy as np
import pytest

from tests import learn_ref as R

pytestmark = pytest.mark.gpu
U = R.U32
B = 256
LENGTHS = [1, 2, 3, 5, 63, 255, 256, 257, 1023, 4095, 4096, 4097, 10_001]
HYPER = dict(lr=2e-3, beta1=0.9, beta2=0.99, eps=1e-8)


@pytest.fixture(scope="module")
def dev():
    from emeans_amd import HipDevice
    d = HipDevice()
    yield d
    d.close()


def _scales(v):
    blocks = -(-v.size // B)
    full = np.zeros(blocks * B)
    full[:v.size] = np.abs(v)
    return full.reshape(blocks, B).max(1) / 448.0


def _by(scale, n):
    return np.repeat(scale, B)[:n]


class Tensor:
    def __init__(self, dev, n, bits, pname, gname, off=0, copy=None, decay=0.01, seed=0):
        import emeans_amd as E
        r = np.random.default_rng(seed + n)
        self.n, self.bits, self.pname, self.gname, self.cname, self.decay = (n, bits, pname, gname,
                                                                             copy, decay)
        m = lambda a, name: R.Padded(dev, a[None], name, 0, off)  # noqa: E731
        self.p, self.g = m(r.standard_normal(n), pname), m(0.1 * r.standard_normal(n), gname)
        self.c = m(np.zeros(n), copy) if copy else None
        self.dev = dev
        if bits == 32:
            self.m, self.v = m(np.zeros(n), "f32"), m(np.zeros(n), "f32")
            self.scales = (None, None)
        else:
            whole = [dev.zeros(n + off, E.F8) for _ in range(2)]
            self.whole = whole
            self.m, self.v = (dev.wrap(w.ptr + off, n, E.F8) for w in whole)
            self.scales = tuple(dev.zeros(-(-n // B), E.F32) for _ in range(2))
        self.desc = E.AdamTensor(self.p.buf if off == 0 else self._cut(self.p, pname),
                                 self._cut(self.g, gname), self._cut(self.m, "f32"),
                                 self._cut(self.v, "f32"), *self.scales,
                                 copy=self._cut(self.c, copy) if copy else None,
                                 weight_decay=decay)
        self.desc.param = self._cut(self.p, pname)

    def _cut(self, pad, name):
        if not isinstance(pad, R.Padded):
            return pad
        return self.dev.wrap(pad.buf.ptr, self.n, R.kind(name))

    def states(self):
        """m, sqrt(v) as the step sees them."""
        if self.bits == 32:
            return self.m.read()[0], np.sqrt(self.v.read()[0])
        got = []
        for b, s in zip((self.m, self.v), self.scales):
            got.append(R.f8_decode(self.dev.read(b)) * _by(self.dev.read(s).astype(float), self.n))
        return got


def _expect(t, p, m, r, step, gscale=1.0):
    g = t.g.value[0] * gscale
    m1 = HYPER["beta1"] * m + (1 - HYPER["beta1"]) * g
    v1 = HYPER["beta2"] * r * r + (1 - HYPER["beta2"]) * g * g
    by = (m1 / (1 - HYPER["beta1"] ** step)) / (
        np.sqrt(v1 / (1 - HYPER["beta2"] ** step)) + HYPER["eps"])
    return p * (1 - HYPER["lr"] * t.decay) - HYPER["lr"] * by, m1, v1, by, g


def _check_step(t, p0, m0, r0, step, gscale=1.0):
    p1, m1, v1, by, g = _expect(t, p0, m0, r0, step, gscale)
    got = t.p.read()[0]
    # m and v: three roundings of each term (the squared root adds two); the
    # quotient a dozen; then p's own two and the type's.
    dm = 4 * U * (np.abs(m0) + np.abs(g))
    dv = 8 * U * v1 + 1e-44
    with np.errstate(divide="ignore", invalid="ignore"):
        rel = np.where(m1 != 0, dm / np.abs(m1), 0) + np.where(v1 > 0, dv / v1, 0) + 16 * U
    tol = 4 * U * np.abs(p0) + HYPER["lr"] * np.abs(by) * rel
    tol = tol + R.UNIT[t.pname] * (np.abs(p1) + tol) * (t.pname != "f32") + R.TINY[t.pname]
    assert np.all(np.abs(got - p1) <= tol), (t.n, t.pname, np.abs(got - p1).max())
    if t.c is not None:
        assert np.all(np.abs(t.c.read()[0] - p1) <= 5 * U * np.abs(p1) + tol
                      + R.UNIT[t.cname] * 1.01 * np.abs(p1) + R.TINY[t.cname])
    if t.bits == 32:
        assert np.all(np.abs(t.m.read()[0] - m1) <= dm)
        assert np.all(np.abs(t.v.read()[0] - v1) <= dv)
        return
    for b, s, want, dw in ((t.m, t.scales[0], m1, dm),
                           (t.v, t.scales[1], np.sqrt(v1), 16 * U * np.sqrt(v1) + 1e-22)):
        scale = t.dev.read(s).astype(float)
        assert np.all(np.abs(scale - _scales(want)) <= _scales(dw) * 448 + 4 * U * scale)
        by = _by(scale, t.n)
        back = R.f8_decode(t.dev.read(b)) * by
        # Half the spacing of the codes: 2^-4 of a value, 2^-10 at the least; a
        # positive root is raised to the least code, 2^-9.
        least = 2.0 ** -10 if want is m1 else 2.0 ** -9
        tol = (2.0 ** -4) * np.abs(want) * 1.001 + least * 1.001 * by + dw
        assert np.all(np.abs(back - want) <= tol)
        if want is not m1:
            assert np.all((back > 0) == (want > 0))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pname,gname", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"),
                                         ("f32", "bf16"), ("bf16", "f32")])
def test_three_steps(dev, bits, pname, gname):
    from emeans_amd import AdamW
    ts = [Tensor(dev, n, bits, pname, gname, copy="bf16" if pname == "f32" and n % 2 else None,
                 decay=0.01 * (n % 3)) for n in LENGTHS]
    plan = AdamW(dev, [t.desc for t in ts])
    for step in (1, 2, 3):
        before = [(t.p.read()[0], *t.states()) for t in ts]
        plan.step(step=step, **HYPER)
        for t, b in zip(ts, before):
            _check_step(t, *b, step)
    plan.close()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_offsets_and_gradient_scale(dev, bits, off):
    from emeans_amd import AdamW
    ts = [Tensor(dev, n, bits, pn, gn, off=off, copy="f16" if pn == "f32" else None)
          for n in (1, 7, 300, 5000) for pn, gn in (("f32", "f16"), ("f16", "bf16"))]
    plan = AdamW(dev, [t.desc for t in ts])
    before = [(t.p.read()[0], *t.states()) for t in ts]
    plan.step(step=1, grad_scale=0.125, **HYPER)
    for t, b in zip(ts, before):
        _check_step(t, *b, 1, 0.125)


def test_blocks_of_zeros_and_wide_ranges(dev):
    """No gradient at all leaves states of zero and only decays the parameters; gradients
    over twelve decades keep the small ones' root off the code zero."""
    from emeans_amd import AdamW
    t = Tensor(dev, 1024, 8, "f32", "f32")
    g = np.zeros(1024)
    g[256:512] = 10.0 ** -np.linspace(0, 12, 256)
    g[512] = 3.0
    t.g = R.Padded(dev, g[None], "f32")
    t.desc.grad = t._cut(t.g, "f32")
    plan = AdamW(dev, [t.desc])
    for step in (1, 2):
        before = (t.p.read()[0], *t.states())
        plan.step(step=step, **HYPER)
        _check_step(t, *before, step)
    assert np.all(np.isfinite(t.p.read()))
    assert dev.read(t.scales[0])[0] == 0.0 and dev.read(t.scales[1])[3] == 0.0


def test_an_element_that_is_not_finite_stays_alone(dev):
    from emeans_amd import AdamW
    for bits in (32, 8):
        t = Tensor(dev, 512, bits, "f32", "f32")
        p0, m0, r0 = (t.p.read()[0], *t.states())
        g = t.g.value[0].copy()
        g[3], g[300] = np.nan, np.inf
        bad = R.Padded(dev, g[None], "f32")
        t.desc.grad = t._cut(bad, "f32")
        AdamW(dev, [t.desc]).step(step=1, **HYPER)
        m, r = t.states()
        rest = np.ones(512, bool)
        rest[[3, 300]] = False
        p1, m1, v1, _, _ = _expect(t, p0, m0, r0, 1)
        assert np.all(np.abs(t.p.read()[0] - p1)[rest] <= 1e-5)
        assert np.isfinite(m[rest]).all() and np.isfinite(r[rest]).all()
        assert np.all(np.abs(m - m1)[rest] <= 2.0 ** -4 * np.abs(m1)[rest] + 1e-3)
        assert np.isnan(m[3]) and not np.isfinite(m[300])


def test_many_tensors_and_none(dev):
    from emeans_amd import AdamW
    ts = [Tensor(dev, 1 + (37 * i) % 900, 32 if i % 2 else 8, "f32", "f32", seed=i)
          for i in range(150)]
    plan = AdamW(dev, [t.desc for t in ts])
    before = [(t.p.read()[0], *t.states()) for t in ts]
    plan.step(step=5, **HYPER)
    for t, b in zip(ts, before):
        _check_step(t, *b, 5)
    AdamW(dev, []).step(step=1, **HYPER)


def test_refusals(dev):
    from emeans_amd import BF16, F16, F32, F8, U32, AdamTensor, AdamW, EmeansHipInvalid

    def refused(*tensors):
        with pytest.raises(EmeansHipInvalid):
            AdamW(dev, list(tensors))

    z = lambda n=600, k=F32: dev.zeros(n, k)  # noqa: E731
    p, g, m, v = z(), z(), z(), z()
    m8, v8, ms, vs = z(600, F8), z(600, F8), z(3), z(3)
    plan = AdamW(dev, [AdamTensor(p, g, m, v)])
    AdamW(dev, [AdamTensor(p, g, m8, v8, ms, vs)])
    refused(AdamTensor(z(k=U32), g, m, v))
    refused(AdamTensor(p, z(k=F8), m, v))
    refused(AdamTensor(p, z(599), m, v))
    refused(AdamTensor(p, g, z(599), v))
    refused(AdamTensor(p, g, z(k=BF16), z(k=BF16)))
    refused(AdamTensor(p, g, m, v8, ms, vs))
    refused(AdamTensor(p, g, m8, v8))                     # no scales
    refused(AdamTensor(p, g, m, v, ms, vs))               # scales of no use
    refused(AdamTensor(p, g, m8, v8, z(2), vs))           # short scales
    refused(AdamTensor(p, g, m8, v8, z(3, F16), vs))
    refused(AdamTensor(p, g, m, v, copy=z()))             # a copy in 32 bits
    refused(AdamTensor(p, g, m, v, copy=z(599, BF16)))
    refused(AdamTensor(p, g, m, m))                       # overlaps
    refused(AdamTensor(p, p, m, v))
    refused(AdamTensor(p, g, m, v), AdamTensor(p, g, z(), z()))
    refused(AdamTensor(p, g, m, v), AdamTensor(dev.wrap(p.ptr + 2396, 600, F32), g, z(), z()))
    refused(AdamTensor(p, g, m, v, weight_decay=float("nan")))
    for bad in (dict(step=0), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1e-8),
                dict(lr=float("inf")), dict(grad_scale=float("nan"))):
        with pytest.raises(EmeansHipInvalid):
            plan.step(**{**HYPER, "step": 1, **bad})
    plan.close()
    with pytest.raises(EmeansHipInvalid):
        plan.step(step=1, **HYPER)
