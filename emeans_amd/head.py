"""A classifier that learns a clustering: rows through a layer norm, a linear layer
with one row of weights for every cluster, softmax cross entropy against the
labels that `assign` or a training gave, AdamW.

    model = Emeans(Config(d=768, k=1024, spherical=True))
    labels = model.train(x).labels
    head = ClusterHead(768, 1024, centroids=model.centroids())
    losses = head.fit(other_view_of_x, labels, epochs=3, batch=16384)

`step` takes resident rows: layer_norm, cross_entropy, cross_entropy_grad,
layer_norm_grad and one AdamW step over all parameters, queued on the device's stream
without a wait. `fit` uploads each batch of host rows, and waits for its losses. With
norm="rms" the norm is rms_norm; with max_norm the gradients count as if clipped to that
global norm, and a step whose gradients are not all finite changes nothing (it counts as a
step all the same).

`answer` gives the likeliest clusters of resident rows, with their log probabilities and the
answers' entropies, in 8 bits: the normalized rows and the classes as codes (rms_norm or
quantize), their product8 in F32, log_probs.

`python -m emeans_amd.head` runs this on synthetic rows.
"""

from dataclasses import dataclass
from typing import List, Optional

import numpy as np

from . import (BF16, F16, F32, F8, MAX_TOP, NONE, U32, AdamTensor, AdamW, Config, DevBuf, Emeans,
               GradNorm, HipDevice, make_assigner)


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


@dataclass
class Answer:
    """What ClusterHead.answer says of n rows: the likeliest clusters (n x top, NONE where there
    are fewer), their log probabilities, the entropies (n), and the log probabilities of the
    given clusters (n; None without them)."""
    ids: np.ndarray
    logp: np.ndarray
    entropy: np.ndarray
    given: Optional[np.ndarray]


class ClusterHead:
    """d: columns of the rows; k: clusters; kind: what rows and the classes' working
    copy are held as (F32, F16 or BF16; the parameters themselves are F32);
    state_bits: 32, or 8 for AdamW states of one byte (rounded at random); centroids: k x d
    initial weights (else small random ones); seed: of both random choices; scale: factor of the logits;
    norm: "layer" (with a bias) or "rms"; max_norm: the gradients' largest global norm (None: any)."""

    EPS = 1e-5
    ANSWER_LOGITS = 1 << 26  # logits that `answer` holds at a time (a row's at least)
    # F16 gradients are those of so many times the loss, and AdamW divides by it. (A mean over
    # 16,384 rows has rows' gradients of 6e-5 of their classes' weights, about F16's least
    # normal number. A class's is at most the scale times its largest element of a
    # normalized row: in range for elements below 64.)
    F16_LOSS_SCALE = 1024.0

    def __init__(self, d: int, k: int, kind: int = F32, state_bits: int = 32, centroids=None,
                 scale: float = 1.0, weight_decay: float = 0.01, seed: int = 1234,
                 dev: Optional[HipDevice] = None, norm: str = "layer",
                 max_norm: Optional[float] = None):
        if d <= 0 or k <= 0:
            raise ValueError("d and k must be positive")
        if kind not in (F32, F16, BF16):
            raise ValueError("kind must be F32, F16 or BF16")
        if state_bits not in (32, 8):
            raise ValueError("state_bits must be 32 or 8")
        if norm not in ("layer", "rms"):
            raise ValueError("norm must be 'layer' or 'rms'")
        if max_norm is not None and not max_norm > 0:
            raise ValueError("max_norm must be positive")
        self.rms, self.max_norm = norm == "rms", max_norm
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
        self.norm_bias = None if self.rms else self.dev.zeros(d, F32)
        # The products read the classes in the rows' kind.
        self._w = self.w if kind == F32 else self.dev.zeros(k * d, kind)
        if kind != F32:
            self.dev.write(self._w, 0, _encode(w, kind).reshape(-1))
        self._dw = self.dev.zeros(k * d, kind)
        self._dweight = self.dev.zeros(d, F32)
        self._dbias = None if self.rms else self.dev.zeros(d, F32)
        copy = None if kind == F32 else self._w
        tensors = [self._tensor(self.w, self._dw, state_bits, weight_decay, copy),
                   self._tensor(self.norm_weight, self._dweight, state_bits, 0.0)]
        if not self.rms:
            tensors.append(self._tensor(self.norm_bias, self._dbias, state_bits, 0.0))
        self._plan = AdamW(self.dev, tensors, seed=int(r.integers(1 << 63)))
        self._norm = None if max_norm is None else GradNorm(self.dev, [t.grad for t in tensors])
        self._clip = None if max_norm is None else self.dev.zeros(2, F32)
        self._rows = 0
        self._frozen = None  # the steps made when the classes' codes were

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
        if self.rms:
            self.dev.rms_norm(x, n, self.d, self.norm_weight, self._y, rstd=self._rstd,
                              eps=self.EPS)
        else:
            self.dev.layer_norm(x, n, self.d, self.norm_weight, self.norm_bias, self._y,
                                self._mean, self._rstd, eps=self.EPS)
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
        if self.rms:
            self.dev.rms_norm_grad(self._dy, x, n, self.d, self.norm_weight, self._rstd, None,
                                   self._dweight)
        else:
            self.dev.layer_norm_grad(self._dy, x, n, self.d, self.norm_weight, self._mean,
                                     self._rstd, None, self._dweight, self._dbias)
        if self._norm is not None:
            self._norm.norm(self._clip, self.max_norm, 1.0 / self.loss_scale)
        self._plan.step(lr, self.steps + 1, grad_scale=1.0 / self.loss_scale, clip=self._clip)
        self.steps += 1  # (a step that was refused is none)
        return self._loss

    def grad_norm(self) -> float:
        """The global norm of the last step's gradients, before they were clipped (max_norm)."""
        if self._clip is None:
            raise ValueError("the head was made without max_norm")
        return float(self.dev.read_f32(self._clip)[0])

    def freeze(self):
        """The classes' codes for `answer`, from the weights as they are. (`answer` does this
        itself after steps; weights written from outside need it.)"""
        blocks = HipDevice.code_blocks
        if self._frozen is None:
            self._w8 = self.dev.zeros(self.k * HipDevice.code_stride(self.d), F8)
            self._w8_scales = self.dev.zeros(blocks(self.k) * blocks(self.d), F32)
        self.dev.quantize(self.w, self.k, self.d, self._w8, self._w8_scales,
                          tile_rows=HipDevice.CODE_BLOCK)
        self._frozen = self.steps

    def answer(self, x: DevBuf, n: int, top: int = 1, labels: Optional[DevBuf] = None) -> Answer:
        """The `top` likeliest clusters of n resident rows, in 8 bits (see the module); labels:
        the clusters whose log probabilities are wanted, NONE for none."""
        if not 1 <= top <= MAX_TOP:
            raise ValueError(f"top must be 1 to {MAX_TOP}")
        if not self.scale > 0:
            raise ValueError("answers need a positive scale")
        if n < 0 or len(x) < n * self.d or (labels is not None and len(labels) < n):
            raise ValueError("x and labels must hold n rows")
        if x.kind != self.kind:
            raise ValueError("x must be of the head's kind")
        if self._frozen != self.steps:
            self.freeze()
        d, k, dev = self.d, self.k, self.dev
        rows = min(n, max(1, self.ANSWER_LOGITS // k))
        stride, blocks = HipDevice.code_stride(d), HipDevice.code_blocks(d)
        codes, scales = dev.zeros(rows * stride, F8), dev.zeros(rows * blocks, F32)
        normed = None if self.rms else dev.zeros(rows * d, self.kind)
        # F32 whatever the head's kind, as in training: in BF16 logits of 256 are 2 apart, and F16
        # ends at 65,504.
        logits = dev.zeros(rows * k, F32)
        ids, logp = dev.zeros(n * top, U32), dev.zeros(n * top, F32)
        lse, entropy = dev.zeros(n, F32), dev.zeros(n, F32)
        given = None if labels is None else dev.zeros(n, F32)
        e = 4 if self.kind == F32 else 2

        def part(b, at, count, size):
            return None if b is None else dev.wrap(b.ptr + at * size, count, b.kind)
        for a in range(0, n, max(rows, 1)):
            m = min(rows, n - a)
            xa = part(x, a * d, m * d, e)
            if self.rms:
                dev.rms_norm(xa, m, d, self.norm_weight, codes, scales=scales, eps=self.EPS)
            else:
                dev.layer_norm(xa, m, d, self.norm_weight, self.norm_bias, normed, eps=self.EPS)
                dev.quantize(normed, m, d, codes, scales)
            dev.product8(codes, scales, m, d, self._w8, self._w8_scales, k, logits)
            dev.log_probs(logits, m, k, part(labels, a, m, 4), part(given, a, m, 4),
                          part(lse, a, m, 4), entropy=part(entropy, a, m, 4), top=top,
                          top_ids=part(ids, a * top, m * top, 4),
                          top_logp=part(logp, a * top, m * top, 4), scale=self.scale)
        return Answer(dev.read_u32(ids).reshape(n, top), dev.read_f32(logp).reshape(n, top),
                      dev.read_f32(entropy), None if given is None else dev.read_f32(given))

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
    head = ClusterHead(128, 64, kind=BF16, state_bits=8, centroids=model.centroids(), dev=dev,
                       norm="rms", max_norm=1.0)
    for e, loss in enumerate(head.fit(view, labels, epochs=4, batch=4096, lr=1e-2)):
        print(f"epoch {e}: mean loss {loss:.4f}", flush=True)
    print(f"norm of the last step's gradients: {head.grad_norm():.4f}")
    best = head.answer(head.rows(view), len(view), top=3, labels=head.labels(labels))
    print(f"answered in 8 bits with their labels: {np.mean(best.ids[:, 0] == labels):.3f} of the "
          f"rows, among three: {np.mean((best.ids == labels[:, None]).any(1)):.3f}; mean log "
          f"probability of the label {best.given.mean():.4f}, mean entropy {best.entropy.mean():.4f}")


if __name__ == "__main__":
    main()
