"""What the tests of the answering and tuning operators share: codes as their
definition makes them, the operators in 64 bits, and a captured graph."""

import ctypes as C

import numpy as np

from tests import learn_ref as R

BLOCK, TOP = 128, 448.0
NONE = 0xFFFFFFFF
# The finite codes' values by magnitude: code i is the i-th.
VALUES = R.F8[:127]


def nearest_codes(q):
    """float32 -> e4m3 codes, to nearest, ties to the even code; what is not finite NaN."""
    q = np.asarray(q, np.float64)
    a = np.abs(q)
    hi = np.searchsorted(VALUES, a).clip(1, 126)
    lo = hi - 1
    dl, dh = a - VALUES[lo], VALUES[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi).astype(np.uint8)
    code = np.where(np.isfinite(q), code, 0x7F).astype(np.uint8)
    return code | np.where(np.signbit(q), 0x80, 0).astype(np.uint8)


def blocks(n):
    return -(-n // BLOCK)


def wide(d):
    return -(-d // 16) * 16


def quantize(x, rows):
    """Codes and scales of float32 values, from the definition."""
    n, d = x.shape
    x = x.astype(np.float32)
    full = np.zeros((-(-n // rows) * rows, blocks(d) * BLOCK), np.float32)
    full[:n, :d] = x
    tiles = full.reshape(-1, rows, blocks(d), BLOCK)
    with np.errstate(all="ignore"):
        mag = np.where(np.isfinite(tiles), np.abs(tiles), np.float32(0))
        scale = (mag.max((1, 3)) / np.float32(TOP)).astype(np.float32)
        s = scale[:, None, :, None]
        q = np.where(s > 0, (tiles / np.where(s > 0, s, np.float32(1))).astype(np.float32), tiles)
    return nearest_codes(q).reshape(full.shape)[:n, :d], scale


def spread(scale, rows, n, d):
    """A scale for every element."""
    return np.repeat(np.repeat(scale.astype(np.float64), rows, 0)[:n], BLOCK, 1)[:, :d]


class CodeBuf:
    """A rows x d matrix of codes in a buffer with a stride and an offset (multiples of 16), the
    rest filled with a code that must neither be read nor change. codes None: an output."""

    def __init__(self, dev, rows, d, codes=None, pad=0, off=0, fill=0x7F):
        from emeans_amd import F8
        self.dev, self.rows, self.d, self.ld, self.off = dev, rows, d, wide(d) + 16 * pad, 16 * off
        self.before = np.full(self.off + rows * self.ld + 16, fill, np.uint8)
        self.at = self.off + (np.arange(rows)[:, None] * self.ld + np.arange(d)[None, :])
        if codes is not None:
            self.before[self.at] = codes
        self.whole = dev.zeros(self.before.size, F8)
        dev.write(self.whole, 0, self.before)
        self.buf = dev.wrap(self.whole.ptr + self.off, self.before.size - self.off, F8)

    def read(self):
        raw = self.dev.read(self.whole)
        tail = self.off + (np.arange(self.rows)[:, None] * self.ld +
                           np.arange(self.d, wide(self.d))[None, :])
        assert not raw[tail].any(), "codes from a row's end to its next multiple of 16"
        outside = np.ones(raw.size, bool)
        outside[self.at] = False
        outside[tail] = False
        assert raw[outside].tobytes() == self.before[outside].tobytes(), "wrote around the codes"
        return raw[self.at]


def rms_norm(h, w, eps):
    rstd = 1.0 / np.sqrt((h * h).mean(1) + eps)
    return h * rstd[:, None] * w, rstd


def rms_norm_grad(dy, dh, h, rstd, w):
    u = h * rstd[:, None]
    g = dy * w
    dx = dh + rstd[:, None] * (g - u * (g * u).mean(1, keepdims=True))
    return dx, (dy * u).sum(0)


class LogProbs:
    """log p, entropies and the order of the classes of rows of logits, in 64 bits."""

    def __init__(self, z, scale=1.0):
        with np.errstate(all="ignore"):
            z = z.astype(np.float64)
            self.z = z * scale
            self.m = self.z.max(1)
            b = np.where(np.isfinite(self.m), self.m, 0.0)[:, None]
            self.d = self.z - b
            e = np.exp(self.d)
            s = e.sum(1)
            self.lse = np.log(s) + b[:, 0]
            self.odd = np.isnan(z).any(1) | np.isposinf(z).any(1)
            self.lse[self.odd] = np.nan
            self.none = np.isneginf(z).all(1)
            self.p = np.where(self.none[:, None], 0.0, e / s[:, None])
            self.lp = np.where(self.none[:, None], -np.inf, self.z - self.lse[:, None])
            self.h = -np.where(self.p > 0, self.p * self.lp, 0.0).sum(1)
            self.h[self.odd] = np.nan
            self.order = np.argsort(-z, axis=1, kind="stable")

    def given(self, tokens):
        has = tokens != NONE
        r = np.arange(len(tokens))
        out = np.where(has, self.lp[r, np.where(has, tokens, 0).astype(np.int64)], 0.0)
        out[self.odd & has] = np.nan
        return out

    def top(self, m):
        n, k = self.z.shape
        ids = np.full((n, m), NONE, np.uint32)
        lp = np.full((n, m), -np.inf)
        c = min(m, k)
        first = self.order[:, :c]
        vals = np.take_along_axis(self.lp, first, 1)
        ids[:, :c] = np.where(np.isneginf(vals), NONE, first)
        lp[:, :c] = vals
        ids[self.odd] = NONE
        lp[self.odd] = np.nan
        return ids, lp

    def grad(self, tokens, gl, gh, scale):
        n, k = self.z.shape
        has = (tokens != NONE) & ~self.none
        gl = np.where(has, gl, 0.0)
        gh = np.where(self.none, 0.0, gh)
        with np.errstate(all="ignore"):
            plp = np.where(self.p > 0, self.p * (self.lp + self.h[:, None]), 0.0)
        dz = -gl[:, None] * self.p - gh[:, None] * plp
        r = np.arange(n)[has]
        dz[r, tokens[has].astype(np.int64)] += gl[has]
        return dz * scale


_HIP = None


def hip():
    global _HIP
    if _HIP is None:
        _HIP = C.CDLL("libamdhip64.so")
        for name in ("hipStreamBeginCapture", "hipStreamEndCapture", "hipGraphInstantiate",
                     "hipGraphLaunch", "hipStreamSynchronize", "hipGraphExecDestroy",
                     "hipGraphDestroy"):
            getattr(_HIP, name).restype = C.c_int
    return _HIP


class Graph:
    """What f queues on dev's stream, captured; replay() runs and waits for it."""

    def __init__(self, dev, f):
        from emeans_amd._lib import lib
        self.stream = C.c_void_p(lib().emh_stream(dev._ctx))
        g, self.exe = C.c_void_p(), C.c_void_p()
        assert hip().hipStreamBeginCapture(self.stream, 2) == 0  # relaxed
        try:
            f()
        finally:
            rc = hip().hipStreamEndCapture(self.stream, C.byref(g))
        assert rc == 0
        assert hip().hipGraphInstantiate(C.byref(self.exe), g, None, None, C.c_size_t(0)) == 0
        assert hip().hipGraphDestroy(g) == 0

    def replay(self):
        assert hip().hipGraphLaunch(self.exe, self.stream) == 0
        assert hip().hipStreamSynchronize(self.stream) == 0

    def close(self):
        assert hip().hipGraphExecDestroy(self.exe) == 0
