"""The answering and tuning operators run together: a head with an RMS norm and clipped
gradients against the same training in 64 bits, its answers in 8 bits against their own
definition, and one chain of all operators, eager and captured."""

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


def _rows(n, d, k, seed):
    r = np.random.default_rng(seed)
    w = r.standard_normal((k, d)) / np.sqrt(d)
    lab = r.integers(0, k, n).astype(np.int32)
    x = 4 * w[lab] + 0.3 * r.standard_normal((n, d))
    lab[::13] = -1
    return x.astype(np.float32), lab, w.astype(np.float32)


@pytest.mark.parametrize("max_norm", [0.05, 100.0])
def test_steps_follow_the_64_bit_training(dev, max_norm):
    """Eight steps in f32 with an RMS norm, clipped always or never: as the layer norm's head,
    1e-3 of the distance moved (a step moves a weight by about lr whatever the gradient's size,
    so errors show where one is near zero)."""
    from emeans_amd.head import ClusterHead
    n, d, k, lr = 2000, 48, 20, 1e-3
    x, lab, w0 = _rows(n, d, k, 1)
    head = ClusterHead(d, k, centroids=w0, dev=dev, norm="rms", max_norm=max_norm)
    assert head.norm_bias is None
    xb, lb = head.rows(x), head.labels(lab)
    u = np.where(lab < 0, A.NONE, lab).astype(np.uint32)
    p = [w0.astype(float), np.ones(d)]
    m, v = [np.zeros_like(a) for a in p], [np.zeros_like(a) for a in p]
    x64, has = x.astype(float), lab >= 0
    for t in range(1, 9):
        loss = dev.read_f32(head.step(xb, lb, n, lr))[:n]
        y, rstd = A.rms_norm(x64, p[1], head.EPS)
        want, _, soft, _ = R.cross_entropy(y, p[0], u, 1.0)
        dy, dw, _ = R.cross_entropy_grad(y, p[0], u, 1.0, soft, np.where(has, 1.0 / has.sum(), 0))
        _, dg = A.rms_norm_grad(dy, 0.0, x64, rstd, p[1])
        norm = np.sqrt((dw ** 2).sum() + (dg ** 2).sum())
        assert abs(head.grad_norm() - norm) <= 1e-4 * norm
        f = min(1.0, max_norm / norm)
        assert (f < 1) == (max_norm < 1)
        for i, g in enumerate((dw * f, dg * f)):
            m[i] = 0.9 * m[i] + 0.1 * g
            v[i] = 0.999 * v[i] + 0.001 * g * g
            by = (m[i] / (1 - 0.9 ** t)) / (np.sqrt(v[i] / (1 - 0.999 ** t)) + 1e-8)
            p[i] = p[i] * (1 - lr * (0.01 if i == 0 else 0.0)) - lr * by
        assert np.abs(loss - want).max() <= 1e-3
    for got, a, start in ((head.w, p[0], w0), (head.norm_weight, p[1], np.ones(d))):
        off = np.abs(dev.read_f32(got).astype(float).reshape(a.shape) - a)
        assert off.mean() <= 0.002 * np.abs(a - start).mean()


def test_a_step_with_gradients_that_are_not_finite_changes_nothing(dev):
    from emeans_amd.head import ClusterHead
    x, lab, w0 = _rows(300, 40, 11, 2)
    head = ClusterHead(40, 11, centroids=w0, dev=dev, norm="rms", max_norm=1.0, state_bits=8)
    lb = head.labels(lab)
    head.step(head.rows(x), lb, 300, 1e-3)
    before = dev.read(head.w).tobytes(), dev.read(head.norm_weight).tobytes()
    bad = x.copy()
    bad[1, 3] = np.inf
    head.step(head.rows(bad), lb, 300, 1e-3)
    assert not np.isfinite(head.grad_norm())
    assert (dev.read(head.w).tobytes(), dev.read(head.norm_weight).tobytes()) == before
    head.step(head.rows(x), lb, 300, 1e-3)
    assert np.isfinite(head.grad_norm()) and np.isfinite(dev.read(head.w)).all()
    assert dev.read(head.w).tobytes() != before[0]


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_answers_are_those_of_the_codes(dev, norm, name):
    """The head's answers against log probabilities of the products of its own codes: logits off
    by a block's roundings (f32) and one of the head's kind."""
    from emeans_amd.head import ClusterHead
    n, d, k, top = 700, 200, 333, 7
    x, lab, w0 = _rows(n, d, k, 5)
    head = ClusterHead(d, k, kind=R.kind(name), centroids=3 * w0, dev=dev, norm=norm, scale=0.7)
    xb, lb = head.rows(x), head.labels(lab)
    head.step(xb, lb, n, 1e-3)
    head.ANSWER_LOGITS = 300 * k  # three blocks of rows
    got = head.answer(xb, n, top, lb)
    # The codes, made as the head makes them.
    q, s = A.CodeBuf(dev, n, d), R.Padded(dev, np.zeros((n, A.blocks(d))), "f32")
    if norm == "rms":
        dev.rms_norm(xb, n, d, head.norm_weight, q.buf, scales=s.buf, eps=head.EPS)
    else:
        y = dev.zeros(n * d, R.kind(name))
        dev.layer_norm(xb, n, d, head.norm_weight, head.norm_bias, y, eps=head.EPS)
        dev.quantize(y, n, d, q.buf, s.buf)
    wq, ws = A.quantize(dev.read_f32(head.w).reshape(k, d), 128)
    a = R.f8_decode(q.read()) * A.spread(s.read(), 1, n, d)
    b = R.f8_decode(wq) * A.spread(ws, 128, k, d)
    z, mag = a @ b.T, np.abs(a) @ np.abs(b).T
    off = (140 * U + (0 if name == "f32" else 7 * 2.0 ** -13)) * mag
    off += R.UNIT[name] * np.abs(z) * 1.01
    worst = 0.7 * off.max(1)
    ref = A.LogProbs(z, 0.7)
    # Every logit moves by at most `worst`, lse too; log probabilities by twice that.
    tol = 2 * worst + 1e-5
    u = np.where(lab < 0, A.NONE, lab).astype(np.uint32)
    assert np.all(np.abs(got.given - ref.given(u)) <= tol)
    assert np.all(np.abs(got.logp - np.take_along_axis(ref.lp, got.ids.astype(int), 1)) <= tol[:, None])
    # None of the classes left out is likelier than the last by more than both may be off.
    left = ref.lp.copy()
    np.put_along_axis(left, got.ids.astype(int), -np.inf, 1)
    assert np.all(left.max(1) <= got.logp[:, -1] + 2 * tol)
    assert np.all(np.diff(got.logp, axis=1) <= 0)
    # An entropy moves by at most sum p |log p + H| times a logit's error twice.
    lh = (ref.p * np.abs(np.where(ref.p > 0, ref.lp, 0) + ref.h[:, None])).sum(1)
    assert np.all(np.abs(got.entropy - ref.h) <= 2 * worst * (lh + worst) * 1.1 + 1e-5)


def test_answers_follow_the_weights(dev):
    from emeans_amd.head import ClusterHead
    x, lab, w0 = _rows(50, 32, 9, 3)
    head = ClusterHead(32, 9, centroids=w0, dev=dev, norm="rms")
    xb = head.rows(x)
    one = head.answer(xb, 50, 9)
    assert one.given is None and np.array_equal(np.sort(one.ids, 1), np.tile(np.arange(9), (50, 1)))
    head.step(xb, head.labels(lab), 50, 0.1)
    two = head.answer(xb, 50, 9)
    assert not np.array_equal(one.logp, two.logp)
    dev.write(head.w, 0, w0.reshape(-1))
    dev.write(head.norm_weight, 0, np.ones(32))
    head.freeze()
    assert np.array_equal(head.answer(xb, 50, 9).logp, one.logp)
    none = head.answer(xb, 0, 2)
    assert none.ids.shape == (0, 2)
    few = head.answer(xb, 3, 12)  # more than there are
    assert (few.ids[:, 9:] == A.NONE).all() and np.isneginf(few.logp[:, 9:]).all()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_answers_of_long_classes(dev, name):
    """Logits of 240,000: whole in f32, of a class that is likelier than all others by
    thousands: its log probability is 0 and so is the entropy."""
    from emeans_amd.head import ClusterHead
    d, k = 64, 5
    x = np.zeros((k, d), np.float32)
    x[np.arange(k), np.arange(k)] = 3.0
    head = ClusterHead(d, k, kind=R.kind(name), centroids=1e4 * x, dev=dev, norm="rms")
    got = head.answer(head.rows(x), k, 1, head.labels(np.arange(k)))
    assert np.array_equal(got.ids[:, 0], np.arange(k))
    assert (got.logp == 0).all() and (got.given == 0).all() and (got.entropy == 0).all()


def test_refusals(dev):
    from emeans_amd.head import ClusterHead
    for bad in (dict(norm="batch"), dict(max_norm=0.0), dict(max_norm=-1.0),
                dict(max_norm=float("nan"))):
        with pytest.raises(ValueError):
            ClusterHead(8, 4, dev=dev, **bad)
    head = ClusterHead(8, 4, dev=dev, scale=-1.0)
    xb = head.rows(np.zeros((3, 8)))
    with pytest.raises(ValueError):
        head.answer(xb, 3)
    with pytest.raises(ValueError):
        head.grad_norm()
    head = ClusterHead(8, 4, dev=dev)
    for bad in (dict(top=0), dict(top=33), dict(n=4), dict(labels=head.labels(np.zeros(2, int)))):
        with pytest.raises(ValueError):
            head.answer(**{**dict(x=xb, n=3), **bad})
    from emeans_amd import BF16, F16
    for other in (F16, BF16):  # rows of another kind than the head's
        with pytest.raises(ValueError, match="kind"):
            head.answer(dev.zeros(24, other), 3)


def test_all_operators_in_one_chain(dev):
    """Rows and residual -> norm in codes -> logits -> answers -> gradient of the logits; norm and
    gradient again in 16 bits; the gradients' norm: eager, and captured and replayed with other
    rows, the eager program's own calls and waits in between."""
    from emeans_amd import BF16, F32, F8, U32, GradNorm, HipDevice
    n, d, k, top = 300, 256, 1000, 4
    r = np.random.default_rng(4)
    x, res = r.standard_normal((n, d)), 0.3 * r.standard_normal((n, d))
    w = r.standard_normal((k, d)) / 16
    tok = r.integers(0, k, n).astype(np.uint32)
    xb, rb, h, y, dz, dy, dx = (dev.zeros(n * c, BF16) for c in (d, d, d, d, k, d, d))
    wb, q, w8 = dev.upload_f32(w), dev.zeros(n * d, F8), dev.zeros(k * d, F8)
    s, ws = dev.zeros(n * 2, F32), dev.zeros(8 * 2, F32)
    z = dev.zeros(n * k, BF16)
    lp, lse, ent, rstd = (dev.zeros(n, F32) for _ in range(4))
    ids, tops, dweight = dev.zeros(n * top, U32), dev.zeros(n * top, F32), dev.zeros(d, F32)
    t, gl, norm = dev.upload_u32(tok), dev.upload_f32(r.standard_normal(n)), dev.zeros(2, F32)
    dev.write(rb, 0, R.encode(res, "bf16").reshape(-1))
    dev.write(dy, 0, R.encode(r.standard_normal((n, d)), "bf16").reshape(-1))
    dev.quantize(wb, k, d, w8, ws, tile_rows=HipDevice.CODE_BLOCK)
    plan = GradNorm(dev, [dz, dx, dweight])

    def chain():
        dev.rms_norm(xb, n, d, None, q, residual=rb, h=h, scales=s)
        dev.product8(q, s, n, d, w8, ws, k, z)
        dev.log_probs(z, n, k, t, lp, lse, entropy=ent, top=top, top_ids=ids, top_logp=tops)
        dev.log_probs_grad(z, n, k, t, lse, dz, entropy=ent, glogp=gl, gentropy=gl)
        dev.rms_norm(h, n, d, None, y, rstd=rstd)
        dev.rms_norm_grad(dy, h, n, d, None, rstd, dx, dweight)
        plan.clip(norm, 1.0)
    outs = (h, q, s, z, lp, lse, ent, ids, tops, dz, y, rstd, dx, dweight, norm)

    def read():
        return [dev.read(b).tobytes() for b in outs]
    graph = None
    for i in range(4):
        dev.write(xb, 0, R.encode(x * (1 + i), "bf16").reshape(-1))
        chain()
        eager = read()
        assert len(set(eager)) == len(outs)
        if graph is None:
            dev.sync()
            graph = A.Graph(dev, chain)
        for b in outs:
            dev.write(b, 0, np.zeros(len(b)))
        dev.sync()
        graph.replay()
        assert read() == eager
        # And they are what they should be: the answers of these logits.
        zv = R.decode(dev.read(z), "bf16").reshape(n, k)
        ref = A.LogProbs(zv)
        assert np.array_equal(dev.read(ids).reshape(n, top), ref.top(top)[0])
        assert np.abs(dev.read(lp) - ref.given(tok)).max() <= 1e-4
    graph.close()


def test_the_example_runs(dev, capsys):
    from emeans_amd import head
    head.main()
    out = capsys.readouterr().out
    assert out.count("epoch") == 4 and "answered in 8 bits" in out
