"""Layer norm and its gradient against 64 bits: every element type, rows held
by a sixteenth of a wave to rows read in pieces, strides and offsets, and
rows that a norm can go wrong on."""

import os
import subprocess
import sys

import numpy as np
import pytest

from tests import learn_ref as R

pytestmark = pytest.mark.gpu
EPS = 1e-5
U = R.U32


@pytest.fixture(scope="module")
def dev():
    from emeans_amd import HipDevice
    d = HipDevice()
    yield d
    d.close()


SIZES = [(1, 1), (1, 2), (3, 5), (7, 64), (16, 384), (33, 300), (5, 1000), (300, 768), (2, 1025),
         (3, 2047), (4, 4096), (5, 4099), (2, 8192), (3, 9001), (1100, 96), (2049, 40), (530, 130)]


def _run(dev, x, name, w, b, wname, pad=0, off=0, dy=None, in_place=False):
    from emeans_amd import F32
    rows, d = x.shape
    px = R.Padded(dev, x, name, pad, off)
    py = px if in_place else R.Padded(dev, np.zeros_like(x), name, 2 * pad, off, fill=7.0)
    pw, pb = (None if v is None else R.Padded(dev, v[None], wname, 0, off) for v in (w, b))
    mean, rstd = (dev.zeros(max(rows, 1), F32) for _ in range(2))
    dev.layer_norm(px.buf, rows, d, pw and pw.buf, pb and pb.buf, py.buf, mean, rstd, eps=EPS,
                   ldx=px.ld, ldy=py.ld)
    got = dict(y=py.read(), mean=dev.read(mean)[:rows].astype(float),
               rstd=dev.read(rstd)[:rows].astype(float),
               w=np.ones(d) if w is None else pw.value[0],
               b=np.zeros(d) if b is None else pb.value[0], x=px.value)
    if dy is not None:
        pd = R.Padded(dev, dy, name, 3 * pad, off)
        po = R.Padded(dev, np.zeros_like(x), name, pad, off, fill=7.0)
        pdw, pdb = (R.Padded(dev, np.zeros((1, d)), wname, 0, off, fill=7.0) for _ in range(2))
        dev.layer_norm_grad(pd.buf, px.buf, rows, d, pw and pw.buf, mean, rstd, po.buf, pdw.buf,
                            pdb.buf, lddy=pd.ld, ldx=px.ld, lddx=po.ld)
        got.update(dx=po.read(), dw=pdw.read()[0], db=pdb.read()[0], dy=pd.value)
    return got


def _check(got, name, wname):
    """A sum of d terms in f32 is off by at most (adds in a chain) u times the
    terms' magnitudes; a lane's chain is at most d / 16 long, and the lanes' and
    waves' joins, the division, the root and the products are within 32 more
    roundings. A result rounded to its type adds that type's unit roundoff."""
    x, w, b = got["x"], got["w"], got["b"]
    rows, d = x.shape
    y, mean, rstd, h = R.layer_norm(x, w, b, EPS)
    K = (d / 16 + 32) * U
    top = np.abs(x).max(1)
    # The mean's error moves every difference by it; rstd's is relative.
    dm = K * top
    dh = (dm * rstd)[:, None] + (K + (dm * rstd) ** 2)[:, None] * (1 + np.abs(h))
    assert np.all(np.abs(got["mean"] - mean) <= dm + 1e-45)
    assert np.all(np.abs(got["rstd"] - rstd) <= rstd * (2 * K + 2 * (dm * rstd) ** 2))
    tol = dh * np.abs(w) + 2 * U * np.abs(b) + R.UNIT[name] * np.abs(y) * 1.01 + R.TINY[name]
    assert np.all(np.abs(got["y"] - y) <= tol)
    if "dx" not in got:
        return
    dy = got["dy"]
    dx, dw, db = R.layer_norm_grad(dy, h, rstd, w)
    u = np.abs(dy * w)
    um, hm, dhm = u.max(1), np.abs(h).max(1), dh.max(1)
    off = rstd * um * (4 * K * (1 + hm) ** 2 + 2 * dhm * (1 + 2 * hm))
    assert np.all(np.abs(got["dx"] - dx) <=
                  off[:, None] + R.UNIT[name] * np.abs(dx) * 1.01 + R.TINY[name])
    # Chains over rows: a group's rows, its workgroup's groups and the workgroups.
    K2 = (rows / 256 + 128) * U
    off = K2 * np.abs(dy * h).sum(0) + (np.abs(dy) * dh).sum(0)
    assert np.all(np.abs(got["dw"] - dw) <= off + R.UNIT[wname] * np.abs(dw) * 1.01 + R.TINY[wname])
    off = K2 * np.abs(dy).sum(0)
    assert np.all(np.abs(got["db"] - db) <= off + R.UNIT[wname] * np.abs(db) * 1.01 + R.TINY[wname])


def _inputs(rows, d, seed):
    r = np.random.default_rng(seed)
    x = r.standard_normal((rows, d)) * (0.5 + r.random((rows, 1))) + r.standard_normal((rows, 1))
    return x, 1 + 0.2 * r.standard_normal(d), 0.2 * r.standard_normal(d), r.standard_normal((rows, d))


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,d", SIZES)
def test_against_64_bits(dev, rows, d, name):
    x, w, b, dy = _inputs(rows, d, rows * 7 + d)
    wname = name if (rows + d) % 2 else "f32"
    _check(_run(dev, x, name, w, b, wname, dy=dy), name, wname)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [17, 300, 1025])
@pytest.mark.parametrize("pad,off", [(0, 1), (3, 0), (5, 3)])
def test_strides_and_offsets(dev, name, d, pad, off):
    x, w, b, dy = _inputs(9, d, d + pad)
    _check(_run(dev, x, name, w, b, name, pad, off, dy), name, name)


@pytest.mark.parametrize("d", [20, 700, 3000, 17000])
def test_without_weight_and_in_place(dev, d):
    x, _, _, dy = _inputs(6, d, d)
    for name in ("f32", "bf16"):
        _check(_run(dev, x, name, None, None, "f32", dy=dy), name, "f32")
        _check(_run(dev, x, name, None, None, "f32", in_place=False), name, "f32")
        got = _run(dev, x, name, None, None, "f32", in_place=True)
        _check(got, name, "f32")


@pytest.mark.parametrize("d", [700, 9001])
def test_dx_over_dy_and_parts_left_out(dev, d):
    from emeans_amd import F32
    x, w, _, dy = _inputs(40, d, d)
    full = _run(dev, x, "f32", w, None, "f32", dy=dy)
    xb, wb = dev.upload_f32(x), dev.upload_f32(w)
    mean, rstd = dev.upload_f32(full["mean"]), dev.upload_f32(full["rstd"])
    for dw, db in ((True, True), (False, True), (False, False)):
        g = dev.upload_f32(dy)
        bw, bb = dev.zeros(d, F32), dev.zeros(d, F32)
        dev.layer_norm_grad(g, xb, 40, d, wb, mean, rstd, g, bw if dw else None, bb if db else None)
        assert np.array_equal(dev.read(g), full["dx"].ravel().astype(np.float32))
        assert np.array_equal(dev.read(bw), (full["dw"] * dw).astype(np.float32))
        assert np.array_equal(dev.read(bb), (full["db"] * db).astype(np.float32))
    bw = dev.zeros(d, F32)
    dev.layer_norm_grad(dev.upload_f32(dy), xb, 40, d, wb, mean, rstd, None, bw, None)
    assert np.array_equal(dev.read(bw), full["dw"].astype(np.float32))


def test_offset_rows_constant_rows_and_rows_that_are_not_finite(dev):
    """A row's mean far beyond its spread, no spread at all, and a row with an
    infinity and one with a NaN, which stay in their rows."""
    d = 512
    x, w, b, dy = _inputs(8, d, 3)
    x[0] += 1000.0
    x[1] = 5.0
    got = _run(dev, x, "f32", w, b, "f32", dy=dy)
    _check(got, "f32", "f32")
    x[5, 7] = np.inf
    x[6, 8] = np.nan
    bad = _run(dev, x, "f32", w, b, "f32", dy=dy)
    rest = [0, 1, 2, 3, 4, 7]
    for what in ("y", "dx"):
        assert np.array_equal(bad[what][rest], got[what][rest])
        assert np.isnan(bad[what][6]).all()
        assert np.isnan(bad[what][5]).any()


def test_gradient_is_the_difference(dev):
    """The gradients along random directions against central differences of
    the 64-bit forward pass: truncation h^2 and cancellation 1e-16 / h leave
    1e-9 of the terms, the f32 gradients 1e-5 of them."""
    rows, d = 12, 333
    x, w, b, dy = _inputs(rows, d, 11)
    got = _run(dev, x, "f32", w, b, "f32", dy=dy)
    x, w, b, dy = got["x"], got["w"], got["b"], got["dy"]
    r = np.random.default_rng(5)
    h = 1e-5

    def total(x, w, b):
        return float((R.layer_norm(x, w, b, EPS)[0] * dy).sum())

    for _ in range(3):
        ex, ew, eb = r.standard_normal(x.shape), r.standard_normal(d), r.standard_normal(d)
        for grad, args, e in ((got["dx"], 0, ex), (got["dw"], 1, ew), (got["db"], 2, eb)):
            up, down = [x, w, b], [x, w, b]
            up[args], down[args] = up[args] + h * e, down[args] - h * e
            diff = (total(*up) - total(*down)) / (2 * h)
            assert abs(float((grad * e).sum()) - diff) <= 1e-5 * float(np.abs(grad * e).sum())


def test_no_rows(dev):
    from emeans_amd import F32
    e, one = dev.zeros(0, F32), dev.upload_f32(np.ones(5))
    dev.layer_norm(e, 0, 5, one, one, e, e, e)
    dw, db = dev.upload_f32(np.ones(5)), dev.upload_f32(np.ones(5))
    dev.layer_norm_grad(e, e, 0, 5, one, e, e, e, dw, db)
    assert not dev.read(dw).any() and not dev.read(db).any()


def test_the_same_bits_every_time(dev):
    x, w, b, dy = _inputs(3000, 200, 2)
    a, c = (_run(dev, x, "bf16", w, b, "f32", dy=dy) for _ in range(2))
    assert all(np.array_equal(a[k], c[k]) for k in a)


TORCH = """
import torch
torch.cuda.init()
from emeans_amd import BF16, F32, HipDevice
from emeans_amd._lib import lib
dev = HipDevice()
mine = torch.cuda.ExternalStream(lib().emh_stream(dev._ctx))
rows, d = 20_000, 640
for seed in range(3):
    x = torch.randn(rows, d, device="cuda")
    for _ in range(20):
        x = x * 1.01 - 0.01
    x = x.to(torch.bfloat16)
    y = torch.empty_like(x)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    mine.wait_stream(torch.cuda.current_stream())
    dev.layer_norm(dev.wrap(x.data_ptr(), x.numel(), BF16), rows, d, None, None,
                   dev.wrap(y.data_ptr(), y.numel(), BF16),
                   dev.wrap(mean.data_ptr(), rows, F32), dev.wrap(rstd.data_ptr(), rows, F32))
    torch.cuda.current_stream().wait_stream(mine)
    f = x.float()
    want = (f - f.mean(1, keepdim=True)) / (f.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt()
    off = (y.float() - want).abs().max()
    assert off <= 2.0 ** -8 * want.abs().max() * 1.01, off
print("streams: ok")
"""


def test_on_torch_tensors_of_another_stream():
    """Inputs that torch's stream is still writing: the context's stream, taken
    up by torch, waits for them and torch for it. In a process of its own:
    torch brings its own HIP runtime, which has to be the first one loaded."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", TORCH], cwd=root, capture_output=True, text=True,
                       timeout=110)
    assert r.returncode == 0 and "streams: ok" in r.stdout, r.stderr[-2000:]


def test_refusals(dev):
    from emeans_amd import BF16, F32, F8, U32, EmeansHipInvalid
    x, v = dev.zeros(60, F32), dev.zeros(10, F32)
    h = dev.zeros(60, BF16)
    y = dev.zeros(60, F32)
    s, t = dev.zeros(6, F32), dev.zeros(6, F32)
    ok = (x, 6, 10, v, v, y, s, t)
    dev.layer_norm(*ok)

    def refused(fn, *a, **k):
        with pytest.raises(EmeansHipInvalid):
            fn(*a, **k)

    def but(i, b):
        return ok[:i] + (b,) + ok[i + 1:]

    n = dev.layer_norm
    refused(n, *but(2, 0))                              # no columns
    refused(n, *but(1, 7))                              # more rows than the buffer holds
    refused(n, *but(1, 2 ** 62))                        # ... by an overflow
    refused(n, *ok, ldx=9)                              # a stride below d
    refused(n, *ok, ldx=11)                             # a stride past the buffer
    refused(n, *but(0, dev.zeros(60, U32)))             # kinds
    refused(n, *but(0, dev.zeros(60, F8)))
    refused(n, *but(5, h))
    refused(n, *but(3, dev.zeros(10, BF16)))            # neither f32 nor x's kind
    refused(n, *but(3, dev.zeros(9, F32)))              # short
    refused(n, *but(6, dev.zeros(5, F32)))
    refused(n, *but(6, dev.zeros(6, BF16)))
    refused(n, *ok, eps=-1.0)
    refused(n, *ok, eps=float("nan"))
    refused(n, *but(5, dev.wrap(x.ptr + 4, 59, F32)), ldx=0)  # over part of x
    refused(n, *but(6, x))                              # statistics over the rows
    refused(n, *but(7, s))                              # and over each other
    refused(n, *but(0, dev.wrap(x.ptr + 2, 60, F32)))   # not at an element
    g = dev.layer_norm_grad
    dy, dx, dw, db = dev.zeros(60, F32), dev.zeros(60, F32), dev.zeros(10, F32), dev.zeros(10, F32)
    ok = (dy, x, 6, 10, v, s, t, dx, dw, db)
    g(*ok)
    refused(g, *but(0, h))
    refused(g, *but(5, dev.zeros(5, F32)))
    refused(g, *but(7, h))
    refused(g, *but(7, x))                              # x is read while dx is written
    refused(g, *but(7, dev.wrap(dy.ptr + 4, 59, F32)))
    refused(g, *but(8, dev.zeros(9, F32)))
    refused(g, *but(8, db))
    refused(g, *but(8, v))
    refused(g, *ok, lddx=9)
    with pytest.raises((EmeansHipInvalid, AttributeError)):
        g(*but(5, None))
