"""A classifier that learns a clustering: rows through a layer norm, a linear layer
with one row of weights for every cluster, softmax cross entropy against the
labels that `assign` or a training gave, AdamW.

    model = Emeans(Config(d=768, k=1024, spherical=True))
    labels = model.train(x).labels
    head = ClusterHead(768, 1024, centroids=model.centroids())
    losses = head.fit(other_view_of_x, labels, epochs=3, batch=16384)

`step` takes resident rows: layer_norm, cross_entropy, cross_entropy_grad,
layer_norm_grad and one AdamW step over all parameters, queued on the device's stream
without a wait. `fit` uploads each batch of host rows, and waits for its losses.

`python -m emeans_amd.head` runs this on synthetic rows.
"""

from typing import List, Optional

import numpy as np

from . import (BF16, F16, F32, F8, NONE, AdamTensor, AdamW, Config, DevBuf, Emeans,
               HipDevice, make_assigner)


def _encode(a, kind):
    """float32 values as a buffer of that kind holds them."""
    a = np.ascontiguousarray(a, np.float32)
    if kind == F32:
        return a
    if kind == F16:
        return a.astype(np.float16)
    b = a.view(np.uint32).astype(np.uint64)  # to nearest, ties to even
    out = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    out[np.isnan(a)] = 0x7FC0
    return out


class ClusterHead:
    """d: columns of the rows; k: clusters; kind: what rows and the classes' working
    copy are held as (F32, F16 or BF16; the parameters themselves are F32);
    state_bits: 32, or 8 for AdamW states of one byte (rounded at random); centroids: k x d
    initial weights (else small random ones); seed: of both random choices; scale: factor of the logits."""

    EPS = 1e-5
    # F16 gradients are those of so many times the loss, and AdamW divides by it. (A mean over
    # 16,384 rows has rows' gradients of 6e-5 of their classes' weights, about F16's least
    # normal number. A class's is at most the scale times its largest element of a
    # normalized row: in range for elements below 64.)
    F16_LOSS_SCALE = 1024.0

    def __init__(self, d: int, k: int, kind: int = F32, state_bits: int = 32, centroids=None,
                 scale: float = 1.0, weight_decay: float = 0.01, seed: int = 1234,
                 dev: Optional[HipDevice] = None):
        if d <= 0 or k <= 0:
            raise ValueError("d and k must be positive")
        if kind not in (F32, F16, BF16):
            raise ValueError("kind must be F32, F16 or BF16")
        if state_bits not in (32, 8):
            raise ValueError("state_bits must be 32 or 8")
        self.d, self.k, self.kind, self.scale, self.steps = d, k, kind, float(scale), 0
        self.loss_scale = self.F16_LOSS_SCALE if kind == F16 else 1.0
        self.dev = dev if dev is not None else make_assigner()
        r = np.random.default_rng(seed)
        if centroids is None:
            w = (r.standard_normal((k, d)) / np.sqrt(d)).astype(np.float32)
        else:
            w = np.ascontiguousarray(centroids, np.float32).reshape(-1)
            if w.size != k * d:
                raise ValueError("centroids must be k x d")
        self.w = self.dev.upload_f32(w)
        self.norm_weight = self.dev.upload_f32(np.ones(d))
        self.norm_bias = self.dev.zeros(d, F32)
        # The products read the classes in the rows' kind.
        self._w = self.w if kind == F32 else self.dev.zeros(k * d, kind)
        if kind != F32:
            self.dev.write(self._w, 0, _encode(w, kind).reshape(-1))
        self._dw = self.dev.zeros(k * d, kind)
        self._dweight, self._dbias = self.dev.zeros(d, F32), self.dev.zeros(d, F32)
        copy = None if kind == F32 else self._w
        self._plan = AdamW(self.dev, [
            self._tensor(self.w, self._dw, state_bits, weight_decay, copy),
            self._tensor(self.norm_weight, self._dweight, state_bits, 0.0),
            self._tensor(self.norm_bias, self._dbias, state_bits, 0.0)],
            seed=int(r.integers(1 << 63)))
        self._rows = 0

    def _tensor(self, param, grad, bits, decay, copy=None):
        n = len(param)
        if bits == 32:
            m, v = (self.dev.zeros(n, F32) for _ in range(2))
            return AdamTensor(param, grad, m, v, copy=copy, weight_decay=decay)
        blocks = -(-n // AdamW.BLOCK)
        m, v = (self.dev.zeros(n, F8) for _ in range(2))
        ms, vs = (self.dev.zeros(blocks, F32) for _ in range(2))
        return AdamTensor(param, grad, m, v, ms, vs, copy, decay)

    def _hold(self, n):
        """Buffers for batches of n rows."""
        if n <= self._rows:
            return
        self._y, self._dy = (self.dev.zeros(n * self.d, self.kind) for _ in range(2))
        self._mean, self._rstd, self._loss, self._lse = (self.dev.zeros(n, F32) for _ in range(4))
        self._rows = n

    def _forward(self, x, labels, n):
        self._hold(n)
        self.dev.layer_norm(x, n, self.d, self.norm_weight, self.norm_bias, self._y, self._mean,
                            self._rstd, eps=self.EPS)
        self.dev.cross_entropy(self._y, n, self.d, self._w, self.k, labels, self._loss, self._lse,
                               scale=self.scale)

    def rows(self, x) -> DevBuf:
        """Host rows (n x d) as a device buffer of the head's kind."""
        raw = _encode(x, self.kind).reshape(-1)
        if raw.size % self.d:
            raise ValueError("x must be n x d")
        b = self.dev.zeros(raw.size, self.kind)
        self.dev.write(b, 0, raw)
        return b

    def labels(self, labels) -> DevBuf:
        """Host labels as a device buffer; negative ones (rows without a cluster) are NONE."""
        a = np.asarray(labels)
        if a.size and a.max() > NONE:
            raise ValueError("a label has more than 32 bits")
        a = np.where(a < 0, NONE, a) if np.issubdtype(a.dtype, np.signedinteger) else a
        return self.dev.upload_u32(a)

    def loss(self, x: DevBuf, labels: DevBuf, n: int) -> np.ndarray:
        """The rows' losses (0 for a row without a label)."""
        self._forward(x, labels, n)
        return self.dev.read_f32(self._loss, (0, n))

    def step(self, x: DevBuf, labels: DevBuf, n: int, lr: float) -> DevBuf:
        """One training step on n resident rows; the buffer that gets their losses."""
        self._forward(x, labels, n)
        self.dev.cross_entropy_grad(self._y, n, self.d, self._w, self.k, labels, self._lse,
                                    self._dy, self._dw, scale=self.scale,
                                    loss_scale=self.loss_scale)
        self.dev.layer_norm_grad(self._dy, x, n, self.d, self.norm_weight, self._mean, self._rstd,
                                 None, self._dweight, self._dbias)
        self._plan.step(lr, self.steps + 1, grad_scale=1.0 / self.loss_scale)
        self.steps += 1  # (a step that was refused is none)
        return self._loss

    def fit(self, x, labels, epochs: int = 1, batch: int = 16384, lr: float = 1e-3,
            seed: int = 0) -> List[float]:
        """Train on host rows (n x d) and their labels; the mean loss of each epoch."""
        x, labels = np.ascontiguousarray(x, np.float32).reshape(-1, self.d), np.asarray(labels)
        n = x.shape[0]
        if labels.shape != (n,):
            raise ValueError("labels must have an entry for every row")
        if batch <= 0:
            raise ValueError("batch must be positive")
        has = labels >= 0 if np.issubdtype(labels.dtype, np.signedinteger) else labels != NONE
        r, out = np.random.default_rng(seed), []
        for _ in range(epochs):
            order, total = r.permutation(n), 0.0
            for a in range(0, n, batch):
                at = order[a:a + batch]
                loss = self.step(self.rows(x[at]), self.labels(labels[at]), at.size, lr)
                total += float(self.dev.read_f32(loss, (0, at.size)).sum(dtype=np.float64))
            out.append(total / max(1, int(has.sum())))
        return out


def main():
    from . import synth
    x, _ = synth.blobs_spherical(20_000, 128, 64, 0.1, seed=7)
    dev = make_assigner()
    model = Emeans(Config(d=128, k=64, spherical=True, seed=7), dev)
    labels = model.train(x).labels
    view = x + 0.05 * np.random.default_rng(1).standard_normal(x.shape).astype(np.float32)
    head = ClusterHead(128, 64, kind=BF16, state_bits=8, centroids=model.centroids(), dev=dev)
    for e, loss in enumerate(head.fit(view, labels, epochs=4, batch=4096, lr=1e-2)):
        print(f"epoch {e}: mean loss {loss:.4f}", flush=True)


if __name__ == "__main__":
    main()
