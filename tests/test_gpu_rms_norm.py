"""RMS norm, its gradient and 8-bit codes against 64 bits: every element type, rows held by a
sixteenth of a wave to rows read in pieces, strides and offsets, results in place, values that
are not finite, graphs."""

import numpy as np
import pytest

from tests import answer_ref as A
from tests import learn_ref as R

pytestmark = pytest.mark.gpu
EPS = 1e-6
U = R.U32
SIZES = [(1, 1), (3, 5), (1, 8), (7, 64), (16, 384), (33, 300), (5, 1000), (300, 768), (2, 1025),
         (3, 2047), (4, 4096), (5, 4099), (2, 8192), (3, 9001), (1100, 96), (2049, 40), (530, 130)]


@pytest.fixture(scope="module")
def dev():
    from emeans_amd import HipDevice
    d = HipDevice()
    yield d
    d.close()


def _inputs(rows, d, seed):
    r = np.random.default_rng(seed)
    x = r.standard_normal((rows, d)) * (0.5 + r.random((rows, 1)))
    return x, 0.3 * r.standard_normal((rows, d)), 1 + 0.1 * r.standard_normal(d), r


def _sum(x, r, name):
    """x + r as the type holds it (the sum in f32 first, as every type's is)."""
    return R.decode(R.encode((x.astype(np.float32) + r.astype(np.float32)), name), name)


def _k(d):
    # Sums: a lane's chain is at most d / 16 long; joins, root, quotient and products are within
    # 32 more roundings.
    return (d / 16 + 32) * U


def _check_y(y, h, w, name):
    want, rstd = A.rms_norm(h, w, EPS)
    tol = 2 * _k(h.shape[1]) * np.abs(want) + R.UNIT[name] * np.abs(want) * 1.01 + R.TINY[name]
    assert np.all(np.abs(y - want) <= tol)
    return rstd


@pytest.mark.parametrize("rows,d", SIZES)
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_forward_and_gradient(dev, rows, d, name):
    from emeans_amd import F32
    x, res, w, r = _inputs(rows, d, rows * 1000 + d)
    i = (rows + d) % 3
    pad, off, wname = [(0, 0, name), (3, 1, "f32"), (1, 5, name)][i]
    px, pr = R.Padded(dev, x, name, pad, off), R.Padded(dev, res, name, 2 * pad, off)
    ph, py = (R.Padded(dev, np.zeros_like(x), name, pad, off, fill=7.0) for _ in range(2))
    pw = R.Padded(dev, w[None], wname, 0, off)
    rstd = dev.zeros(rows, F32)
    dev.rms_norm(px.buf, rows, d, pw.buf, py.buf, residual=pr.buf, h=ph.buf, rstd=rstd, eps=EPS,
                 ldx=px.ld, ldr=pr.ld, ldh=ph.ld, ldy=py.ld)
    h = ph.read()
    assert np.array_equal(h, _sum(px.value, pr.value, name))
    want = _check_y(py.read(), h, pw.value[0], name)
    got = dev.read(rstd).astype(np.float64)
    assert np.all(np.abs(got - want) <= 2 * _k(d) * want)

    dy, dh = (r.standard_normal((rows, d)) for _ in range(2))
    pd, pe = R.Padded(dev, dy, name, pad, off), R.Padded(dev, dh, name, 2 * pad, off)
    po = R.Padded(dev, np.zeros_like(x), name, 2 * pad, off, fill=7.0)
    pg = R.Padded(dev, np.zeros((1, d)), wname, 0, off, fill=7.0)
    dev.rms_norm_grad(pd.buf, ph.buf, rows, d, pw.buf, rstd, po.buf, pg.buf, dh=pe.buf,
                      lddy=pd.ld, ldh=ph.ld, lddx=po.ld, lddh=pe.ld)
    dx, dw = A.rms_norm_grad(pd.value, pe.value, h, want, pw.value[0])
    g = np.abs(pd.value * pw.value[0])
    u = np.abs(h) * want[:, None]
    off = want[:, None] * (g + u * (g * u).mean(1, keepdims=True))
    tol = 8 * _k(d) * off + 2 * U * np.abs(pe.value) + R.UNIT[name] * np.abs(dx) * 1.01 + R.TINY[name]
    assert np.all(np.abs(po.read() - dx) <= tol)
    # Chains over rows: a group's rows, its workgroup's groups and the workgroups.
    tol = ((rows / 16 + 128) * U + 2 * _k(d)) * (np.abs(pd.value) * u).sum(0)
    assert np.all(np.abs(pg.read()[0] - dw) <= tol + R.UNIT[wname] * np.abs(dw) * 1.01 + R.TINY[wname])


@pytest.mark.parametrize("rows,d", SIZES)
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_codes(dev, rows, d, name):
    x, res, w, _ = _inputs(rows, d, rows * 7 + d)
    x[rows // 2] = 0.0
    res[rows // 2] = 0.0
    pad = (rows + d) % 2
    px, pr = R.Padded(dev, x, name, pad, pad), R.Padded(dev, res, name, 0, pad)
    ph = R.Padded(dev, np.zeros_like(x), name, pad, pad, fill=7.0)
    pw = R.Padded(dev, w[None], "f32")
    q = A.CodeBuf(dev, rows, d, pad=pad, off=pad, fill=0x55)
    s = R.Padded(dev, np.zeros((rows, A.blocks(d))), "f32", pad, pad, fill=7.0)
    dev.rms_norm(px.buf, rows, d, pw.buf, q.buf, residual=pr.buf, h=ph.buf, scales=s.buf, eps=EPS,
                 ldx=px.ld, ldr=pr.ld, ldh=ph.ld, ldy=q.ld, lds=s.ld)
    h = ph.read()
    assert np.array_equal(h, _sum(px.value, pr.value, name))
    y, _ = A.rms_norm(h, pw.value[0], EPS)
    got, scale = R.f8_decode(q.read()), s.read()
    full = np.zeros((rows, A.blocks(d) * 128))
    full[:, :d] = np.abs(y)
    want = full.reshape(rows, -1, 128).max(2) / 448
    rel = 2 * _k(d) + 2 * U
    assert np.all(np.abs(scale - want) <= rel * want)
    # The nearest code of y / scale, both of which may be off by that: half a step (2^-4 of the
    # value, or 2^-10), and what the quotient's own error moves.
    sc = A.spread(scale, 1, rows, d)
    tol = np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10 * sc) * (1 + 1e-3) + 2 * rel * np.abs(y)
    assert np.all(np.abs(got * sc - y) <= tol)
    assert not got[rows // 2].any()


@pytest.mark.parametrize("name,d", [("bf16", 768), ("f16", 300), ("f32", 77), ("bf16", 9001)])
def test_in_place_and_without_what_is_optional(dev, name, d):
    rows = 37
    x, res, w, r = _inputs(rows, d, d)
    # h in the residual's place, y in x's.
    px, pr = R.Padded(dev, x, name), R.Padded(dev, res, name)
    hv = _sum(px.value, pr.value, name)
    dev.rms_norm(px.buf, rows, d, None, px.buf, residual=pr.buf, h=pr.buf, eps=EPS)
    assert np.array_equal(pr.read(), hv)
    rstd = _check_y(px.read(), hv, np.ones(d), name)
    # No residual, no h: y in x's place.
    px = R.Padded(dev, x, name)
    v = px.value
    dev.rms_norm(px.buf, rows, d, None, px.buf, eps=EPS)
    _check_y(px.read(), v, np.ones(d), name)
    # dx in dh's place; dx alone; dweight alone.
    from emeans_amd import F32
    rb = dev.zeros(rows, F32)
    dev.write(rb, 0, rstd.astype(np.float32))
    dy, dh = r.standard_normal((rows, d)), r.standard_normal((rows, d))
    pd, pe = R.Padded(dev, dy, name), R.Padded(dev, dh, name)
    po, pg = R.Padded(dev, dy, name), R.Padded(dev, np.zeros((1, d)), "f32")
    dev.rms_norm_grad(pd.buf, pr.buf, rows, d, None, rb, po.buf, pg.buf, dh=pe.buf)
    dev.rms_norm_grad(pd.buf, pr.buf, rows, d, None, rb, pe.buf, None, dh=pe.buf)
    assert np.array_equal(pe.read(), po.read())
    p2 = R.Padded(dev, np.zeros((1, d)), "f32")
    dev.rms_norm_grad(pd.buf, pr.buf, rows, d, None, rb, None, p2.buf)
    assert np.array_equal(p2.read(), pg.read())
    # Without dh it is zero.
    dev.rms_norm_grad(pd.buf, pr.buf, rows, d, None, rb, pd.buf)
    dx, _ = A.rms_norm_grad(R.Padded(dev, dy, name).value, 0.0, hv, rstd, np.ones(d))
    tol = 64 * _k(d) * np.abs(dx).max() + R.UNIT[name] * np.abs(dx) * 1.01 + R.TINY[name]
    assert np.all(np.abs(pd.read() - dx) <= tol)


def test_gradient_against_differences(dev):
    from emeans_amd import F32
    rows, d, step = 3, 20, 1e-4
    x, _, w, r = _inputs(rows, d, 5)
    dy, dh = r.standard_normal((rows, d)), r.standard_normal((rows, d))
    x32 = x.astype(np.float32).astype(np.float64)
    f = lambda x, w: (dy * A.rms_norm(x, w, EPS)[0]).sum() + (dh * x).sum()  # noqa: E731
    b = {k: R.Padded(dev, v, "f32") for k, v in
         dict(x=x32, w=w[None], dy=dy, dh=dh, y=x32, dx=x32, dw=w[None]).items()}
    rstd = dev.zeros(rows, F32)
    dev.rms_norm(b["x"].buf, rows, d, b["w"].buf, b["y"].buf, rstd=rstd, eps=EPS)
    dev.rms_norm_grad(b["dy"].buf, b["x"].buf, rows, d, b["w"].buf, rstd, b["dx"].buf,
                      b["dw"].buf, dh=b["dh"].buf)
    for got, at, which in ((b["dx"].read(), x32, 0), (b["dw"].read(), w[None], 1)):
        for i in np.ndindex(at.shape):
            e = np.zeros(at.shape)
            e[i] = step
            hi, lo = (f(x32 + s * e, w) if which == 0 else f(x32, w + s * e[0]) for s in (1, -1))
            # Differences: step^2 times a third derivative (below 100 here) and 64-bit rounding.
            assert abs(got[i] - (hi - lo) / (2 * step)) <= 100 * step ** 2 + 1e-9 + 2e-5


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,d", [(1, 1), (1, 16), (5, 300), (130, 128), (129, 257), (257, 1000),
                                    (3, 5000), (1000, 24)])
@pytest.mark.parametrize("tile_rows", [1, 128])
def test_quantize_is_exact(dev, name, rows, d, tile_rows):
    r = np.random.default_rng(rows + d)
    x = r.standard_normal((rows, d)) * np.exp(4 * r.standard_normal((rows, 1)))
    x[rows // 2, d // 2:] = 0.0
    if rows > 3:
        x[3, 0], x[2, d - 1] = np.inf, np.nan
    pad = (rows + d) % 3
    px = R.Padded(dev, x, name, pad, pad)
    q = A.CodeBuf(dev, rows, d, pad=pad, off=pad, fill=0x55)
    srows = rows if tile_rows == 1 else A.blocks(rows)
    s = R.Padded(dev, np.zeros((srows, A.blocks(d))), "f32", pad, pad, fill=7.0)
    dev.quantize(px.buf, rows, d, q.buf, s.buf, tile_rows=tile_rows, ldx=px.ld, ldq=q.ld, lds=s.ld)
    codes, scale = A.quantize(px.value, tile_rows)
    assert np.array_equal(s.read().astype(np.float32), scale)
    got = q.read()
    nan = (codes & 0x7F) == 0x7F
    assert np.array_equal((got & 0x7F) == 0x7F, nan)
    assert np.array_equal(got[~nan], codes[~nan])


@pytest.mark.parametrize("scale", [1e-42, 1e-36, 1e36])
def test_quantize_of_tiny_and_huge_blocks(dev, scale):
    x = (np.random.default_rng(1).standard_normal((4, 200)) * scale).astype(np.float32)
    px, q = R.Padded(dev, x, "f32"), A.CodeBuf(dev, 4, 200)
    s = R.Padded(dev, np.zeros((4, 2)), "f32")
    dev.quantize(px.buf, 4, 200, q.buf, s.buf)
    codes, want = A.quantize(px.value, 1)
    assert np.array_equal(s.read().astype(np.float32), want)
    assert np.array_equal(q.read(), codes)


@pytest.mark.parametrize("d", [300, 9001])
def test_rows_that_are_not_finite_stay_their_own(dev, d):
    rows = 6
    x, _, w, _ = _inputs(rows, d, 3)
    x[1, 3], x[4, d - 1] = np.nan, np.inf
    px, py = R.Padded(dev, x, "bf16"), R.Padded(dev, x, "bf16")
    q, s = A.CodeBuf(dev, rows, d), R.Padded(dev, np.zeros((rows, A.blocks(d))), "f32")
    dev.rms_norm(px.buf, rows, d, None, py.buf, eps=EPS)
    dev.rms_norm(px.buf, rows, d, None, q.buf, scales=s.buf, eps=EPS)
    y, got, sc = py.read(), R.f8_decode(q.read()), s.read()
    fine = [0, 2, 3, 5]
    _check_y(y[fine], px.value[fine], np.ones(d), "bf16")
    assert np.isnan(y[1]).all() and np.isnan(y[4, d - 1])
    assert np.isfinite(got[fine]).all() and np.isnan(got[1]).all() and np.isnan(got[4, d - 1])
    assert np.isfinite(sc).all()


def test_no_rows(dev):
    from emeans_amd import F32
    b, g = dev.zeros(0, F32), R.Padded(dev, np.ones((1, 9)), "f32")
    dev.rms_norm(b, 0, 9, None, dev.zeros(0, F32))
    dev.rms_norm_grad(b, b, 0, 9, None, b, dev.zeros(0, F32), g.buf)
    assert not g.read().any()


def test_refusals(dev):
    from emeans_amd import BF16, F16, F32, F8, U32, EmeansHipInvalid
    x, y, b, u = dev.zeros(100, F32), dev.zeros(100, F32), dev.zeros(100, BF16), dev.zeros(100, U32)
    q, s, f = dev.zeros(320, F8), dev.zeros(20, F32), dev.zeros(10, F32)

    def no(match, call, *args, **kw):
        with pytest.raises(EmeansHipInvalid, match=match):
            call(*args, **kw)
    n = dev.rms_norm
    no("d must be", n, x, 10, 0, None, y)
    no("x must be", n, u, 10, 10, None, y)
    no("x: the buffer's", n, x, 11, 10, None, y)
    no("x: the row stride", n, x, 10, 10, None, y, ldx=9)
    no("residual must be", n, x, 10, 10, None, y, residual=b)
    no("h must be", n, x, 10, 10, None, y, h=b)
    no("y must be", n, x, 10, 10, None, b)
    no("an f8 y comes with scales", n, x, 10, 10, None, q)
    no("an f8 y comes with scales", n, x, 10, 10, None, y, scales=s)
    no("weight must be", n, x, 10, 10, dev.zeros(10, F16), y)
    no("weight: the buffer's", n, x, 10, 10, dev.zeros(9, F32), y)
    no("eps must be", n, x, 10, 10, None, y, eps=-1.0)
    no("eps must be", n, x, 10, 10, None, y, eps=float("nan"))
    no("y overlaps h", n, x, 10, 10, None, y, h=y)
    no("rstd overlaps x", n, x, 10, 10, None, y, rstd=x)
    no("h overlaps x in part", n, x, 9, 10, None, y, h=dev.wrap(x.ptr + 4, 99, F32))
    no("y overlaps x in part", n, x, 5, 10, None, x, ldy=11)
    no("multiple of 16", n, x, 10, 10, None, q, scales=s, ldy=24)
    no("multiple of 16 bytes", n, x, 10, 10, None, dev.wrap(q.ptr + 8, 200, F8), scales=s)
    no("y: the buffer's", n, x, 10, 10, None, dev.zeros(159, F8), scales=s)
    no("scales: the buffer's", n, x, 10, 10, None, q, scales=dev.zeros(9, F32))
    g = dev.rms_norm_grad
    no("dy must be", g, b, x, 10, 10, None, f, y)
    no("rstd must be", g, y, x, 10, 10, None, b, dev.zeros(100, F32))
    no("dx overlaps h", g, y, x, 10, 10, None, f, x)
    no("dweight overlaps dx", g, x, y, 5, 10, None, f, dev.wrap(s.ptr, 20, F32) and
       dev.wrap(q.ptr, 60, F32), dev.wrap(q.ptr, 10, F32))
    no("dh must be", g, y, x, 10, 10, None, f, None, f, dh=b)
    z = dev.quantize
    no("a scale serves", z, x, 10, 10, q, s, tile_rows=2)
    no("q must be", z, x, 10, 10, y, s)
    no("q overlaps", z, x, 5, 10, dev.wrap(x.ptr, 400, F8), s)
    no("scales must be", z, x, 10, 10, q, u)


def test_a_captured_norm_replays(dev):
    from emeans_amd import F32, HipDevice, EmeansHipInvalid
    rows, d = 300, 200
    x, _, w, r = _inputs(rows, d, 11)
    b = {k: R.Padded(dev, v, "bf16") for k, v in dict(x=x, y=x, dy=x, dx=x).items()}
    rstd, dw = dev.zeros(rows, F32), dev.zeros(d, F32)

    def call():
        dev.rms_norm(b["x"].buf, rows, d, None, b["y"].buf, rstd=rstd, eps=EPS)
        dev.rms_norm_grad(b["dy"].buf, b["x"].buf, rows, d, None, rstd, b["dx"].buf, dw)
    call()
    dev.sync()
    g = A.Graph(dev, call)
    # A larger call in between takes a larger workspace; the graph's own stays.
    big = R.Padded(dev, np.ones((4000, 600)), "bf16")
    bw, br = dev.zeros(600, F32), dev.zeros(4000, F32)
    for i in range(4):
        v = R.encode(x * (i + 1), "bf16").reshape(-1)
        dev.write(b["x"].buf, 0, v)
        dev.rms_norm_grad(big.buf, big.buf, 4000, 600, None, br, None, bw)
        dev.sync()
        g.replay()
        got = [dev.read(v.buf).tobytes() for v in (b["y"], b["dx"])] + [dev.read(dw).tobytes()]
        call()
        assert got == [dev.read(v.buf).tobytes() for v in (b["y"], b["dx"])] + [dev.read(dw).tobytes()]
    g.close()
    # A first call may not be captured: its workspace does not exist yet. (One of few rows, which
    # takes none, may.)
    new = HipDevice()
    xb, yb, rb, wb = new.zeros(60000, F32), new.zeros(60000, F32), new.zeros(300, F32), new.zeros(200, F32)
    new.sync()
    with pytest.raises(EmeansHipInvalid, match="before the capture"):
        A.Graph(new, lambda: new.rms_norm_grad(xb, yb, 300, 200, None, rb, None, wb))
    A.Graph(new, lambda: new.rms_norm_grad(xb, yb, 5, 200, None, rb, None, wb)).close()
    new.rms_norm_grad(xb, yb, 300, 200, None, rb, None, wb)
    new.sync()
    new.close()
