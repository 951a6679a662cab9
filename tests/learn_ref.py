"""What the learning operators' tests share: element types as numpy holds them,
and the operators in 64 bits, written from their definitions."""

import numpy as np

U32 = 2.0 ** -24                                  # unit roundoffs
UNIT = {"f32": U32, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}


def kind(name):
    import emeans_amd as E
    return {"f32": E.F32, "f16": E.F16, "bf16": E.BF16}[name]


def bf16_bits(a):
    """float32 -> bfloat16 bits, to nearest, ties to even."""
    b = np.ascontiguousarray(a, np.float32).view(np.uint32).astype(np.uint64)
    out = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    nan = np.isnan(a)
    out[nan] = 0x7FC0
    return out


def encode(a, name):
    """What a buffer of that kind holds of a."""
    a = np.asarray(a, np.float32)
    if name == "f32":
        return a.copy()
    if name == "f16":
        with np.errstate(over="ignore"):
            return a.astype(np.float16)
    return bf16_bits(a)


def decode(raw, name):
    """Its values, in 64 bits."""
    if name == "bf16":
        return (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return raw.astype(np.float64)


# The values of the e4m3 codes 0 .. 127 (the upper half is their negatives).
F8 = np.array([(m / 8.0) * 2.0 ** -6 if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7)
               for e in range(16) for m in range(8)])
F8[127] = np.nan


def f8_decode(raw):
    return np.where(raw & 0x80, -1.0, 1.0) * F8[raw & 0x7F]


class Padded:
    """A rows x d matrix as a buffer with a row stride and an offset, the rest
    filled with a value that must neither be read nor change."""

    def __init__(self, dev, a, name, pad=0, off=0, fill=np.nan):
        rows, d = a.shape
        self.rows, self.d, self.ld, self.off, self.name = rows, d, d + pad, off, name
        full = np.full(off + rows * self.ld + 3, fill, np.float32)
        self.at = off + (np.arange(rows)[:, None] * self.ld + np.arange(d)[None, :])
        full[self.at] = a
        raw = encode(full, name)
        self.before = raw.copy()
        self.whole = dev.zeros(raw.size, kind(name))
        dev.write(self.whole, 0, raw)
        self.dev = dev
        e = raw.itemsize
        self.buf = dev.wrap(self.whole.ptr + off * e, raw.size - off, kind(name))
        self.value = decode(raw[self.at], name)

    def read(self):
        """The matrix now; everything around it as it was."""
        raw = self.dev.read(self.whole)
        outside = np.ones(raw.size, bool)
        outside[self.at] = False
        assert raw[outside].tobytes() == self.before[outside].tobytes(), "wrote around the matrix"
        return decode(raw[self.at], self.name)


def layer_norm(x, w, b, eps):
    mean = x.mean(1)
    o = x - mean[:, None]
    rstd = 1.0 / np.sqrt((o * o).mean(1) + eps)
    h = o * rstd[:, None]
    return h * w + b, mean, rstd, h


def layer_norm_grad(dy, h, rstd, w):
    u = dy * w
    dx = rstd[:, None] * (u - u.mean(1, keepdims=True) - h * (u * h).mean(1, keepdims=True))
    return dx, (dy * h).sum(0), dy.sum(0)


def cross_entropy(x, w, labels, scale):
    """loss, lse and p (the softmax)."""
    z = scale * (x @ w.T)
    top = z.max(1, keepdims=True)
    e = np.exp(z - top)
    s = e.sum(1, keepdims=True)
    lse = (np.log(s) + top)[:, 0]
    has = labels != 0xFFFFFFFF
    at = np.where(has, labels, 0).astype(np.int64)
    loss = np.where(has, lse - z[np.arange(len(z)), at], 0.0)
    return loss, lse, e / s, z


def cross_entropy_grad(x, w, labels, scale, p, up):
    has = labels != 0xFFFFFFFF
    g = p.copy()
    r = np.arange(len(p))[has]
    g[r, labels[has].astype(np.int64)] -= 1.0
    g *= (scale * np.where(has, up, 0.0))[:, None]
    g[~has] = 0.0
    xs = np.where(has[:, None], x, 0.0)
    return g @ w, g.T @ xs, g
