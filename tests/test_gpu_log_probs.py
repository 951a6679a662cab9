"""Log probabilities, entropies and the likeliest classes of rows of logits, and the logits'
gradient, against 64 bits: short rows and long ones that several workgroups share, every type,
addresses, masks, ties, values that are not finite, graphs."""

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


def _inputs(n, k, seed, masks=True):
    r = np.random.default_rng(seed)
    z = 3 * r.standard_normal((n, k))
    z[np.arange(n), r.integers(0, k, n)] += 10 * r.random(n)
    if masks:
        z[(r.random((n, k)) < 0.3) & (r.random((n, 1)) < 0.5)] = -np.inf
        if n > 4:
            z[n // 2] = -np.inf
    tokens = r.integers(0, k, n).astype(np.uint32)
    tokens[r.random(n) < 0.2] = A.NONE
    return z, tokens, r


def _tols(ref, k, tokens):
    """A term exp(d), d = z - m, is off by 2 |d| + 4 roundings of itself (the difference, the
    product by log2 e, and the power, within two units); a lane adds at most k / 64 + 32 terms,
    and 32 more join lanes, waves and parts, each with a factor of its own."""
    K = k / 64 + 96
    d = np.where(ref.p > 0, np.abs(ref.d), 0.0)
    ed, ed2 = (ref.p * d).sum(1), (ref.p * d * d).sum(1)
    ds = U * (K + 2 * ed + 8)                       # log S, absolutely
    m = np.where(np.isfinite(ref.m), np.abs(ref.m), 0.0)
    lse = ds + 2 * U * (m + np.abs(np.where(ref.none, 0, ref.lse)))
    # E / S: the sums' relative errors, and each term's.
    h = ds + U * (2 * (K + 8) * ed + 2 * ed2) + U * (K + 2 * ed + 8) * ed + 4 * U * (ed + 1)
    t = np.where(tokens != A.NONE, tokens, 0).astype(np.int64)
    dt = np.abs(ref.d[np.arange(len(t)), t])
    logp = ds + 2 * U * (np.where(np.isfinite(dt), dt, 0) + m) + 4 * U
    return ds, lse, h, logp


def _near(got, want, tol):
    with np.errstate(invalid="ignore"):
        same = (got == want) | (np.isnan(got) & np.isnan(want)) | (np.abs(got - want) <= tol)
    assert np.all(same), (got[~same][:5], want[~same][:5])


def _run(dev, z, tokens, name, top=0, scale=1.0, pad=0, off=0, entropy=True):
    from emeans_amd import F32, U32
    n, k = z.shape
    pz = R.Padded(dev, z, name, pad, off)
    out = {x: dev.zeros(n, F32) for x in ("logp", "lse", "h")}
    ids, tops = dev.zeros(n * top, U32), dev.zeros(n * top, F32)
    dev.log_probs(pz.buf, n, k, dev.upload_u32(tokens), out["logp"], out["lse"],
                  entropy=out["h"] if entropy else None, top=top, top_ids=ids if top else None,
                  top_logp=tops if top else None, scale=scale, ldz=pz.ld)
    ref = A.LogProbs(pz.value, scale)
    ds, tl, th, tp = _tols(ref, k, tokens)
    got = {x: dev.read(v).astype(np.float64) for x, v in out.items()}
    _near(got["lse"], ref.lse, tl)
    if entropy:
        _near(got["h"], ref.h, th)
    _near(got["logp"], ref.given(tokens), tp)
    if top:
        wi, wl = ref.top(top)
        assert np.array_equal(dev.read(ids).reshape(n, top), wi)
        tol = (ds[:, None] + 2 * U * np.where(np.isfinite(wl), np.abs(wl), 0) +
               2 * U * np.where(np.isfinite(ref.m), np.abs(ref.m), 0)[:, None] * 2 + 4 * U)
        _near(dev.read(tops).reshape(n, top).astype(np.float64), wl, tol + ds[:, None])
    return pz, ref, out, (tl, th)


SIZES = [(1, 1), (1, 2), (3, 7), (5, 64), (300, 65), (2000, 16), (700, 100), (260, 1000),
         (400, 1023), (257, 2048), (300, 4100), (64, 5000), (9, 8191), (2, 40001), (1, 131071),
         (3, 70000)]


@pytest.mark.parametrize("n,k", SIZES)
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_forward(dev, n, k, name):
    z, tokens, _ = _inputs(n, k, n + k)
    i = (n + k) % 4
    top = [0, 1, 8, 32][i] if name != "bf16" else [5, 16, 2, 1][i]
    _run(dev, z, tokens, name, top, scale=[1.0, 0.7, 2.5, 1.0][i], pad=[0, 1, 3, 0][i],
         off=[0, 1, 2, 5][i], entropy=i != 2)


@pytest.mark.parametrize("n,k", [(1, 1), (3, 7), (300, 65), (260, 1000), (40, 4100), (2, 40001)])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_gradient(dev, n, k, name):
    from emeans_amd import F32
    z, tokens, r = _inputs(n, k, 3 * n + k)
    scale, off = (1.0, 0) if n % 2 else (1.7, 3)
    pz, ref, out, (tl, th) = _run(dev, z, tokens, name, scale=scale, pad=off, off=off)
    gl, gh = r.standard_normal(n).astype(np.float32), r.standard_normal(n).astype(np.float32)
    bl, bh, tok = dev.upload_f32(gl), dev.upload_f32(gh), dev.upload_u32(tokens)
    lse, h = out["lse"], out["h"]
    lp = np.where(ref.p > 0, ref.lp, 0.0)
    perr = tl[:, None] + U * (2 * np.abs(lp) + 8)
    for which in ("both", "logp", "entropy", "in place"):
        a = gl if which != "entropy" else 0 * gl
        b = gh if which != "logp" else 0 * gh
        po = pz if which == "in place" else R.Padded(dev, 0 * np.nan_to_num(z), name, 2 * off, off, fill=7.0)
        dev.log_probs_grad(pz.buf, n, k, tok if which != "entropy" else None, lse, po.buf,
                           entropy=h if which != "logp" else None,
                           glogp=bl if which != "entropy" else None,
                           gentropy=bh if which != "logp" else None, scale=scale, ldz=pz.ld,
                           lddz=po.ld)
        want = ref.grad(tokens, a.astype(np.float64), b.astype(np.float64), scale)
        lh = np.abs(lp + ref.h[:, None])
        g = ref.p * (np.abs(a)[:, None] + np.abs(b)[:, None] * lh) * scale
        tol = (perr * g + np.abs(b)[:, None] * ref.p * scale *
               (th[:, None] + tl[:, None] + 4 * U * (np.abs(lp) + np.abs(ref.h)[:, None])) +
               8 * U * (g + np.abs(want) + scale * np.abs(a)[:, None] * (ref.p > 0)))
        _near(po.read(), want, tol + R.UNIT[name] * np.abs(want) * 1.01 + R.TINY[name] + 1e-37)


def test_gradient_against_differences(dev):
    from emeans_amd import F32
    n, k, step = 4, 9, 1e-4
    z, _, r = _inputs(n, k, 8, masks=False)
    tokens = np.array([3, 0, A.NONE, 8], np.uint32)
    z = z.astype(np.float32).astype(np.float64)
    gl, gh = r.standard_normal(n), r.standard_normal(n)

    def f(z):
        ref = A.LogProbs(z, 0.8)
        return (gl * ref.given(tokens)).sum() + (gh * ref.h).sum()
    pz, po = R.Padded(dev, z, "f32"), R.Padded(dev, z, "f32")
    b = [dev.zeros(n, F32) for _ in range(3)]
    t = dev.upload_u32(tokens)
    dev.log_probs(pz.buf, n, k, t, b[0], b[1], entropy=b[2], scale=0.8)
    dev.log_probs_grad(pz.buf, n, k, t, b[1], po.buf, entropy=b[2], glogp=dev.upload_f32(gl),
                       gentropy=dev.upload_f32(gh), scale=0.8)
    got = po.read()
    for i in np.ndindex(n, k):
        e = np.zeros((n, k))
        e[i] = step
        # Differences: step^2 times a third derivative (below 100 here); f32 elsewhere.
        assert abs(got[i] - (f(z + e) - f(z - e)) / (2 * step)) <= 100 * step ** 2 + 1e-5


@pytest.mark.parametrize("n,k", [(3, 5), (300, 1000), (300, 3000), (2, 30000)])
@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_ties_go_to_the_lower_class(dev, n, k, name):
    r = np.random.default_rng(k)
    # Three values alone; one value alone; rising and falling runs.
    _run(dev, r.integers(0, 3, (n, k)).astype(float), np.zeros(n, np.uint32), name, 32)
    _run(dev, np.full((n, k), -2.5), np.zeros(n, np.uint32), name, 32)
    rise = np.floor(np.arange(k) / 7) * np.ones((n, 1)) / 64
    _run(dev, rise, np.zeros(n, np.uint32), name, 20)
    _run(dev, -rise, np.zeros(n, np.uint32), name, 20)
    _run(dev, np.where(r.random((n, k)) < 0.5, 0.0, -0.0), np.zeros(n, np.uint32), name, 9)


@pytest.mark.parametrize("n,k", [(8, 40), (300, 900), (8, 20000)])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_rows_with_few_classes_and_values_that_are_not_finite(dev, n, k, name):
    from emeans_amd import F32
    r = np.random.default_rng(n)
    z = 2 * r.standard_normal((n, k))
    z[0] = -np.inf
    z[1] = -np.inf
    z[1, k - 1] = -3.0        # one class
    z[2] = -np.inf
    z[2, [3, 7, k // 2]] = 1.0
    z[3, 5] = np.nan
    z[4, k - 2] = np.inf
    z[5] = np.nan
    z[6, k // 3] = 60000.0 if name == "f16" else 1e30
    tokens = np.full(n, 5, np.uint32)
    tokens[1] = k - 1
    tokens[7] = A.NONE
    pz, ref, out, _ = _run(dev, z, tokens, name, 6)
    h = dev.read(out["h"])
    assert h[0] == 0 and h[1] == 0 and np.isnan(h[3:6]).all()
    one = dev.upload_f32(np.ones(n))
    po = R.Padded(dev, np.zeros((n, k)), name, fill=7.0)
    dev.log_probs_grad(pz.buf, n, k, dev.upload_u32(tokens), out["lse"], po.buf, entropy=out["h"],
                       glogp=one, gentropy=one)
    g = po.read()
    assert not g[0].any() and not g[1].any() and np.isfinite(g[[0, 1, 2, 6, 7]]).all()
    assert np.isnan(g[3:6]).all()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("k", [40, 9000])
def test_masks_of_the_lowest_value(dev, name, k):
    """Masked by the type's lowest value, and by twice it through the scale: infinite in f32 and
    bf16, where a class has no probability then, and not in f16. Rows: all masked; all but two."""
    from emeans_amd import F32, U32
    low = {"f32": np.finfo(np.float32).min, "f16": -65504.0, "bf16": -(2.0 - 2.0 ** -7) * 2.0 ** 127}[name]
    z = np.full((2, k), low)
    z[1, [3, k - 2]] = 1.0, 2.0
    p, t = R.Padded(dev, z, name), dev.upload_u32(np.array([7, k - 2], np.uint32))
    out = [dev.zeros(c, F32) for c in (2, 2, 2, 8)] + [dev.zeros(8, U32)]
    one, dz = dev.upload_f32(np.ones(2)), R.Padded(dev, 0 * z, name)
    for scale in (1.0, 2.0):
        dev.log_probs(p.buf, 2, k, t, out[0], out[1], entropy=out[2], top=4, top_logp=out[3],
                      top_ids=out[4], scale=scale)
        lp, lse, h, tops, ids = (dev.read(o) for o in out)
        none = scale == 2 and name != "f16"
        if none:
            assert np.isneginf([lp[0], lse[0]]).all() and h[0] == 0
            assert (ids[:4] == A.NONE).all() and np.isneginf(tops[:4]).all()
        else:  # all alike
            assert np.allclose([lp[0], -h[0], *tops[:4]], -np.log(k), rtol=1e-6)
            assert np.array_equal(ids[:4], [0, 1, 2, 3])
        q = 1 / (1 + np.exp(-scale))
        assert np.allclose([lp[1], *tops[4:6]], np.log([q, q, 1 - q]), rtol=1e-6)
        assert np.allclose(h[1], -q * np.log(q) - (1 - q) * np.log(1 - q), rtol=1e-6)
        assert np.array_equal(ids[4:], [k - 2, 3] + ([A.NONE] * 2 if none else [0, 1]))
        dev.log_probs_grad(p.buf, 2, k, t, out[1], dz.buf, entropy=out[2], glogp=one,
                           gentropy=one, scale=scale)
        g = dz.read()
        assert (g[1, [c for c in range(k) if c not in (3, k - 2)]] == 0).all()
        assert np.isfinite(g).all() and (not none or (g[0] == 0).all())


def test_a_class_out_of_range_is_an_error(dev):
    from emeans_amd import F32, EmeansHipInvalid
    z, tokens, _ = _inputs(5, 30, 1, masks=False)
    tokens[:] = 3
    tokens[2] = 30
    pz, po, t = R.Padded(dev, z, "f32"), R.Padded(dev, z, "f32"), dev.upload_u32(tokens)
    lp, lse = dev.zeros(5, F32), dev.zeros(5, F32)
    dev.log_probs(pz.buf, 5, 30, t, lp, lse)
    with pytest.raises(EmeansHipInvalid, match="label out of range"):
        dev.sync()
    got = dev.read(lp)
    assert got[2] == 0 and (got[[0, 1, 3, 4]] < 0).all()
    dev.log_probs_grad(pz.buf, 5, 30, t, lse, po.buf, glogp=dev.upload_f32(np.ones(5)))
    with pytest.raises(EmeansHipInvalid, match="label out of range"):
        dev.sync()
    assert not po.read()[2].any()


@pytest.mark.parametrize("n,k,top", [(1, 131071, 32), (5, 40001, 3), (70, 9000, 8), (400, 5000, 1)])
def test_rows_in_parts_give_the_same_every_time(dev, n, k, top):
    """Whichever of a row's parts is done last: with equal logits in all of them."""
    from emeans_amd import BF16, F32, U32
    z = np.random.default_rng(n).integers(-3, 3, (n, k)).astype(np.float32)
    b, t = dev.zeros(n * k, BF16), dev.upload_u32(np.arange(n).astype(np.uint32))
    dev.write(b, 0, R.encode(z, "bf16").reshape(-1))
    out = [dev.zeros(n, F32) for _ in range(3)] + [dev.zeros(n * top, F32), dev.zeros(n * top, U32)]
    ref, first = A.LogProbs(z), None
    for _ in range(40):
        dev.log_probs(b, n, k, t, out[0], out[1], entropy=out[2], top=top, top_logp=out[3],
                      top_ids=out[4])
        got = [dev.read(o).tobytes() for o in out]
        first = first or got
        assert got == first
    assert np.array_equal(dev.read(out[4]).reshape(n, top), ref.top(top)[0])


def test_gradient_in_place_without_strides(dev):
    from emeans_amd import F32
    n, k = 5, 40
    z, t = np.random.default_rng(9).standard_normal((n, k)), np.arange(n, dtype=np.uint32)
    a, b, lp, lse = dev.upload_f32(z), dev.zeros(n * k, F32), dev.zeros(n, F32), dev.zeros(n, F32)
    one = dev.upload_f32(np.ones(n))
    dev.log_probs(a, n, k, dev.upload_u32(t), lp, lse)
    for to, kw in ((b, {}), (a, {}), (a, dict(ldz=k)), (a, dict(lddz=k))):
        dev.write(a, 0, z.reshape(-1))
        dev.log_probs_grad(a, n, k, dev.upload_u32(t), lse, to, glogp=one, **kw)
        assert dev.read(to).tobytes() == dev.read(b).tobytes() and dev.read(to).any()


def test_no_rows_and_refusals(dev):
    from emeans_amd import F16, F32, U32, EmeansHipInvalid
    z, f, u = dev.zeros(200, F32), dev.zeros(10, F32), dev.zeros(10, U32)
    f2, f3 = dev.zeros(10, F32), dev.zeros(10, F32)
    ids, tops = dev.zeros(40, U32), dev.zeros(40, F32)
    dev.log_probs(z, 0, 20, u, f, f2)
    dev.log_probs_grad(z, 0, 20, u, f, z, glogp=f2)

    def no(match, *args, **kw):
        with pytest.raises(EmeansHipInvalid, match=match):
            dev.log_probs(*args, **kw)
    no("k must be", z, 10, 0, u, f, f2)
    no("z must be", u, 10, 1, u, f, f2)
    no("z: the buffer's", z, 11, 20, None, None, dev.zeros(11, F32))
    no("tokens must be", z, 10, 20, f3, f, f2)
    no("tokens and logp", z, 10, 20, None, f, f2)
    no("tokens and logp", z, 10, 20, u, None, f2)
    no("scale must be", z, 10, 20, u, f, f2, scale=0.0)
    no("scale must be", z, 10, 20, u, f, f2, scale=-1.0)
    no("scale must be", z, 10, 20, u, f, f2, scale=float("inf"))
    no("top must be", z, 10, 20, u, f, f2, top=33, top_ids=dev.zeros(330, U32))
    no("top and its outputs", z, 10, 20, u, f, f2, top=4)
    no("top and its outputs", z, 10, 20, u, f, f2, top_ids=ids)
    no("top_ids must be", z, 10, 20, u, f, f2, top=4, top_ids=tops)
    no("top_ids: the buffer's", z, 10, 20, u, f, f2, top=5, top_ids=ids)
    no("lse must be", z, 10, 20, u, f, u)
    no("logp overlaps lse", z, 10, 20, u, f, f)
    no("overlaps z", z, 10, 20, u, f, z)

    def nog(match, *args, **kw):
        with pytest.raises(EmeansHipInvalid, match=match):
            dev.log_probs_grad(*args, **kw)
    dz = dev.zeros(200, F32)
    nog("dz must be", z, 10, 20, u, f, dev.zeros(200, F16), glogp=f2)
    nog("tokens and glogp", z, 10, 20, u, f, dz)
    nog("entropy and gentropy", z, 10, 20, u, f, dz, glogp=f2, gentropy=f3)
    nog("dz overlaps z in part", z, 5, 20, u, f, z, glogp=f2, lddz=21)
    nog("dz overlaps lse", z, 1, 10, u, f, f, glogp=f2)


@pytest.mark.parametrize("n,k", [(300, 500), (3, 50000)])
def test_a_captured_call_replays(dev, n, k):
    from emeans_amd import F32, U32
    z, tokens, r = _inputs(n, k, 4)
    pz, po = R.Padded(dev, z, "bf16"), R.Padded(dev, np.zeros((n, k)), "bf16")
    t, gl = dev.upload_u32(tokens), dev.upload_f32(r.standard_normal(n))
    lp, lse, h = (dev.zeros(n, F32) for _ in range(3))
    ids = dev.zeros(n * 7, U32)

    def call():
        dev.log_probs(pz.buf, n, k, t, lp, lse, entropy=h, top=7, top_ids=ids)
        dev.log_probs_grad(pz.buf, n, k, t, lse, po.buf, entropy=h, glogp=gl, gentropy=gl)
    call()
    dev.sync()
    g = A.Graph(dev, call)
    outs = (lp, lse, h, ids, po.buf)
    big = R.Padded(dev, np.zeros((4, 300000)), "bf16")
    bl, bi = dev.zeros(4, F32), dev.zeros(4 * 32, U32)
    for i in range(4):
        dev.write(pz.buf, 0, R.encode(z * (1 + i), "bf16").reshape(-1))
        dev.log_probs(big.buf, 4, 300000, None, None, bl, top=32, top_ids=bi)
        dev.sync()
        g.replay()
        got = [dev.read(b).tobytes() for b in outs]
        call()
        assert got == [dev.read(b).tobytes() for b in outs]
    g.close()


def test_two_contexts_at_once(dev):
    """Rows in parts on two contexts, queued in turns without a wait: each has counters and
    parts of its own. A first call may not be captured: they do not exist yet."""
    from emeans_amd import BF16, F32, U32, EmeansHipInvalid, HipDevice
    n, k, top = 40, 30000, 8
    other = HipDevice()
    z = np.random.default_rng(8).standard_normal((2, n, k))
    b = []
    for d, v in zip((dev, other), z):
        o = dict(z=d.zeros(n * k, BF16), lse=d.zeros(n, F32), h=d.zeros(n, F32),
                 ids=d.zeros(n * top, U32))
        d.write(o["z"], 0, R.encode(v, "bf16").reshape(-1))
        d.sync()
        b.append(o)
    call = lambda d, o: d.log_probs(o["z"], n, k, None, None, o["lse"], entropy=o["h"],  # noqa: E731
                                    top=top, top_ids=o["ids"])
    with pytest.raises(EmeansHipInvalid, match="before the capture"):
        A.Graph(other, lambda: call(other, b[1]))
    for _ in range(20):
        for d, o in zip((dev, other), b):
            call(d, o)
    for d, o, v in zip((dev, other), b, z):
        ref = A.LogProbs(R.decode(R.encode(v, "bf16"), "bf16"))
        assert np.array_equal(d.read(o["ids"]).reshape(n, top), ref.top(top)[0])
        assert np.abs(d.read(o["lse"]) - ref.lse).max() <= 1e-5 * np.abs(ref.lse).max()
        assert np.abs(d.read(o["h"]) - ref.h).max() <= 1e-5 * ref.h.max()
    other.close()
