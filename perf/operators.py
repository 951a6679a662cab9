"""The operators of a training step on cluster labels, as measured cases.

One case is a dict; its "kind" says which operator runs:

  loss   HipDevice.cross_entropy: the loss and the log of the softmax's sum
  train  the loss, then HipDevice.cross_entropy_grad: both gradients of its mean
  norm   HipDevice.layer_norm: the rows and their statistics
  ntrain the same, then HipDevice.layer_norm_grad: the gradients of rows, weight and bias
  adamw  AdamW.step over a list of tensors, states in 32 bits or in 8

Inputs and outputs have the case's "type"; losses, statistics and the
gradients of a norm's weight and bias are float32. 8-bit states are held as
float8_e4m3fn codes and a float32 scale for every 256 of them.
"""

import math

import torch

own = False

NONE = -1          # a row without a label (0xFFFFFFFF)
BLOCK = 256        # elements that share the scale of their 8-bit states
TOP = 448.0        # the largest float8_e4m3fn
LEAST = 2.0 ** -9  # the smallest positive one
EPS_NORM = 1e-5
LR, BETA1, BETA2, EPS, STEP, DECAY = 1e-3, 0.9, 0.999, 1e-8, 10, 0.01
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_DEV = []


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # A few new photos scored against a coarse codebook: latency and launches.
        dict(name="loss_16x384_k256_f32", kind="loss", n=16, d=384, k=256, type="f32"),
        # One row against a large codebook: reading the classes once.
        dict(name="loss_1x1024_k16384_bf16", kind="loss", n=1, d=1024, k=16384, type="bf16"),
        # Odd sizes everywhere, in the framework's own type.
        dict(name="train_10007x300_k1000_f32", kind="train", n=10007, d=300, k=1000, type="f32"),
        # One batch of the headline clustering's rows and clusters.
        dict(name="train_16384x768_k1024_bf16", kind="train", n=16384, d=768, k=1024,
             type="bf16"),
        # A large vocabulary, one class short of a round number.
        dict(name="train_8192x1024_k131071_bf16", kind="train", n=8192, d=1024, k=131071,
             type="bf16"),
        # The few rows of the first case through the norm.
        dict(name="norm_16x384_f32", kind="norm", n=16, d=384, type="f32"),
        # Odd rows in half precision.
        dict(name="ntrain_10007x300_f16", kind="ntrain", n=10007, d=300, type="f16"),
        # The headline batch.
        dict(name="ntrain_16384x768_bf16", kind="ntrain", n=16384, d=768, type="bf16"),
        # All rows of the headline data set at once.
        dict(name="ntrain_200000x768_f32", kind="ntrain", n=200_000, d=768, type="f32"),
        # The parameters of a small head: its classes and the norm before it.
        dict(name="adamw_256x384_f32", kind="adamw", k=256, d=384, layers=1, type="f32", bits=32),
        # A codebook of odd size and a dozen norms, the states in 8 bits.
        dict(name="adamw_1000x300_8bit", kind="adamw", k=1000, d=300, layers=12, type="f32",
             bits=8),
        # The large vocabulary's parameters in bfloat16, the states in 8 bits.
        dict(name="adamw_131071x1024_8bit_bf16", kind="adamw", k=131071, d=1024, layers=2,
             type="bf16", bits=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _dim(rng):
    """Mostly the widths that embeddings have, one in four any width."""
    if rng.random() < 0.25:
        return rng.randint(16, 1100)
    return rng.choice([64, 96, 100, 128, 200, 256, 300, 384, 512, 640, 768, 1024])


def draw(rng):
    kind = rng.choice(["loss", "train", "train", "norm", "ntrain", "adamw"])
    d, type_ = _dim(rng), rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind == "loss":
        return dict(kind=kind, n=_log(rng, 1, 16_384), d=d, k=_log(rng, 16, 65_536), type=type_)
    if kind == "train":
        n, k = _log(rng, 16, 16_384), _log(rng, 16, 131_071)
        while n * k * d * (3 if type_ == "f32" else 1) > 8192 * 131_071 * 1024:
            n, k = (n + 1) // 2, (k + 1) // 2
        return dict(kind=kind, n=n, d=d, k=k, type=type_)
    if kind in ("norm", "ntrain"):
        return dict(kind=kind, n=_log(rng, 1, 100_000), d=d, type=type_)
    return dict(kind=kind, k=_log(rng, 16, 32_768), d=d, layers=rng.randint(1, 24),
                type=rng.choice(["f32", "bf16"]), bits=rng.choice([32, 8]))


# ----------------------------------------------------------------- the inputs
def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(1_000_003 * int(seed) + salt)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _inputs(case, seed):
    """The case's tensors, from the seed alone."""
    kind, d, type_ = case["kind"], case["d"], TYPES[case["type"]]
    g = _gen(seed, 1)
    if kind in ("loss", "train"):
        n, k = case["n"], case["k"]
        # Classes as a codebook's rows, unevenly used; rows after a norm, part
        # noise and part their class, so that some are settled and some not; one
        # row in fifty has no label.
        w = _randn(g, k, d).div_(math.sqrt(d))
        weight = torch.arange(1, k + 1, device="cuda", dtype=torch.float32).pow_(-0.7)
        labels = torch.multinomial(weight, n, replacement=True, generator=g)
        x = _randn(g, n, d).add_(w[labels] * 8.0 * torch.rand(n, 1, generator=g, device="cuda"))
        labels[torch.rand(n, generator=g, device="cuda") < 0.02] = NONE
        return dict(x=x.to(type_), w=w.to(type_), labels=labels.to(torch.int32))
    if kind in ("norm", "ntrain"):
        n = case["n"]
        # Rows with an offset and a size of their own.
        x = _randn(g, n, d).mul_(0.5 + torch.rand(n, 1, generator=g, device="cuda"))
        x.add_(_randn(g, n, 1))
        t = dict(x=x.to(type_), weight=_randn(g, d).mul_(0.1).add_(1.0).to(type_),
                 bias=_randn(g, d).mul_(0.1).to(type_))
        if kind == "ntrain":
            t["dy"] = _randn(g, n, d).mul_(1.0 / n).to(type_)
        return t
    # The tensors are pieces of one buffer each, as a program keeps them that
    # saves or reduces them at once; the states are as ten steps leave them.
    _, total = _pieces(case)
    t = dict(p=_randn(g, total).mul_(0.05).to(type_), g=_randn(g, total).mul_(1e-3).to(type_))
    m, v = _randn(g, total).mul_(3e-4), _randn(g, total).square_().mul_(1e-8)
    if case["bits"] == 32:
        return dict(t, m=m, v=v)
    t["m"], t["ms"] = _coded(m)
    t["v"], t["vs"] = _coded(v.sqrt(), LEAST)
    return t


def _pieces(case):
    """(start, length) of every tensor of an adamw case, and the buffers'
    length; a tensor begins at a multiple of BLOCK."""
    at, got = 0, []
    for length in [case["k"] * case["d"]] + [case["d"]] * (2 * case["layers"]):
        got.append((at, length))
        at += (length + BLOCK - 1) // BLOCK * BLOCK
    return got, at


def _split(case, t):
    """The tensors of an adamw case, as views: a list of dicts."""
    return [{name: v[a // BLOCK:(a + length + BLOCK - 1) // BLOCK] if name in ("ms", "vs")
             else v[a:a + length] for name, v in t.items()} for a, length in _pieces(case)[0]]


def _coded(a, least=0.0):
    """Codes and scales of a: every BLOCK values share their largest magnitude
    / TOP, and a positive value's code is at least `least`."""
    blocks = (a.numel() + BLOCK - 1) // BLOCK
    full = torch.nn.functional.pad(a, (0, blocks * BLOCK - a.numel())).view(blocks, BLOCK)
    scale = full.abs().amax(1) / TOP
    q = full / torch.where(scale > 0, scale, torch.ones_like(scale))[:, None]
    q = torch.where((q < least) & (full > 0), torch.full_like(q, least), q)
    return q.clamp_(-TOP, TOP).view(-1)[:a.numel()].to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    t = _inputs(case, seed)
    s = dict(case=dict(case), t=t)
    if own:
        s["own"] = _handles(case, t)
    torch.cuda.synchronize()
    return s


def _handles(case, t):
    """The views, outputs and plan that a program makes once."""
    import emeans_amd as E
    if not _DEV:
        _DEV.append(E.HipDevice(0))
    dev = _DEV[0]
    kinds = {torch.float32: E.F32, torch.int32: E.U32, torch.float16: E.F16,
             torch.bfloat16: E.BF16, torch.float8_e4m3fn: E.F8}
    wrap = lambda v: dev.wrap(v.data_ptr(), v.numel(), kinds[v.dtype])  # noqa: E731
    if case["kind"] == "adamw":
        views = [{name: wrap(v) for name, v in one.items()} for one in _split(case, t)]
        plan = E.AdamW(dev, [
            E.AdamTensor(v["p"], v["g"], v["m"], v["v"], m_scale=v.get("ms"),
                         v_scale=v.get("vs"), weight_decay=DECAY) for v in views])
        return dict(plan=plan, out={name: v for name, v in t.items() if name != "g"})
    f = lambda *shape: torch.zeros(*shape, device="cuda")  # noqa: E731
    n, d = case["n"], case["d"]
    if case["kind"] in ("loss", "train"):
        out = dict(loss=f(n), lse=f(n))
        if case["kind"] == "train":
            out.update(dx=torch.zeros_like(t["x"]), dw=torch.zeros_like(t["w"]))
    else:
        out = dict(y=torch.zeros_like(t["x"]), mean=f(n), rstd=f(n))
        if case["kind"] == "ntrain":
            out.update(dx=torch.zeros_like(t["x"]), dweight=f(d), dbias=f(d))
    return dict(dev=dev, out=out, **{"b_" + k: wrap(v) for k, v in {**t, **out}.items()})


# ---------------------------------------------------------------- the one pass
def run(s):
    return _run_own(s["case"], s["own"]) if own else _PLAIN[s["case"]["kind"]](s["case"], s["t"])


def _run_own(case, o):
    kind = case["kind"]
    if kind == "adamw":
        o["plan"].step(LR, STEP, beta1=BETA1, beta2=BETA2, eps=EPS)
        return o["out"]
    dev, n, d = o["dev"], case["n"], case["d"]
    if kind in ("loss", "train"):
        dev.cross_entropy(o["b_x"], n, d, o["b_w"], case["k"], o["b_labels"], o["b_loss"],
                          o["b_lse"])
        if kind == "train":
            dev.cross_entropy_grad(o["b_x"], n, d, o["b_w"], case["k"], o["b_labels"], o["b_lse"],
                                   o["b_dx"], o["b_dw"])
        return o["out"]
    dev.layer_norm(o["b_x"], n, d, o["b_weight"], o["b_bias"], o["b_y"], o["b_mean"], o["b_rstd"],
                   eps=EPS_NORM)
    if kind == "ntrain":
        dev.layer_norm_grad(o["b_dy"], o["b_x"], n, d, o["b_weight"], o["b_mean"], o["b_rstd"],
                            o["b_dx"], o["b_dweight"], o["b_dbias"])
    return o["out"]


def _plain_loss(case, t):
    return _cross_entropy(t)[0]


def _cross_entropy(t):
    x, w, labels = t["x"].float(), t["w"].float(), t["labels"].long()
    z = x @ w.t()
    top = z.amax(1, keepdim=True)
    lse = (z - top).exp().sum(1).log() + top[:, 0]
    counts = labels >= 0
    at = labels.clamp(min=0)[:, None]
    loss = torch.where(counts, lse - z.gather(1, at)[:, 0], torch.zeros_like(lse))
    return dict(loss=loss, lse=lse), x, w, z, at, counts


def _plain_train(case, t):
    out, x, w, z, at, counts = _cross_entropy(t)
    g = (z - out["lse"][:, None]).exp()
    g.scatter_add_(1, at, torch.full_like(at, -1, dtype=g.dtype))
    g = g * (counts / counts.sum().clamp(min=1))[:, None]
    out["dx"] = (g @ w).to(t["x"].dtype)
    out["dw"] = (g.t() @ x).to(t["w"].dtype)
    return out


def _layer_norm(t):
    x = t["x"].float()
    mean = x.mean(1)
    off = x - mean[:, None]
    rstd = 1.0 / (off.square().mean(1) + EPS_NORM).sqrt()
    h = off * rstd[:, None]
    y = (h * t["weight"].float() + t["bias"].float()).to(t["x"].dtype)
    return dict(y=y, mean=mean, rstd=rstd), h


def _plain_norm(case, t):
    return _layer_norm(t)[0]


def _plain_ntrain(case, t):
    out, h = _layer_norm(t)
    dy = t["dy"].float()
    g = dy * t["weight"].float()
    dx = g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True)
    out["dx"] = (dx * out["rstd"][:, None]).to(t["x"].dtype)
    out["dweight"] = (dy * h).sum(0)
    out["dbias"] = dy.sum(0)
    return out


def _plain_adamw(case, t):
    step = _adamw if case["bits"] == 32 else _adamw8
    for views in _split(case, t):
        step(**views)
    return {name: v for name, v in t.items() if name != "g"}


def _adamw(p, g, m, v):
    g = g.float()
    m.copy_(BETA1 * m + (1.0 - BETA1) * g)
    v.copy_(BETA2 * v + (1.0 - BETA2) * g * g)
    by = (m / (1.0 - BETA1 ** STEP)) / ((v / (1.0 - BETA2 ** STEP)).sqrt() + EPS)
    p.copy_(p.float() * (1.0 - LR * DECAY) - LR * by)


def _adamw8(p, g, m, ms, v, vs):
    n = p.numel()
    m32 = m.float() * ms.repeat_interleave(BLOCK)[:n]
    r = v.float() * vs.repeat_interleave(BLOCK)[:n]
    v32 = r * r
    _adamw(p, g, m32, v32)
    q, scale = _coded(m32)
    m.copy_(q), ms.copy_(scale)
    q, scale = _coded(v32.sqrt(), LEAST)
    v.copy_(q), vs.copy_(scale)


_PLAIN = dict(loss=_plain_loss, train=_plain_train, norm=_plain_norm, ntrain=_plain_ntrain,
              adamw=_plain_adamw)


# ---------------------------------------------------- its size and its answer
def work(case):
    kind, d = case["kind"], case["d"]
    e = 4 if case["type"] == "f32" else 2
    if kind == "adamw":
        count = (case["k"] + 2 * case["layers"]) * d
        # Parameter read and written, gradient read, both states read and written.
        state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        return {"bytes": count * (3 * e + state), "flops": 15 * count}
    n = case["n"]
    if kind in ("norm", "ntrain"):
        # The backward pass is a call of its own and reads the rows again.
        each = 2 if kind == "norm" else 5
        return {"bytes": each * n * d * e + 8 * n + (2 * d * e if kind == "norm" else 8 * d),
                "flops": (8 if kind == "norm" else 20) * n * d}
    k = case["k"]
    each = 1 if kind == "loss" else 2
    return {"bytes": each * (n + k) * d * e + 12 * n,
            "flops": (2 if kind == "loss" else 6) * n * k * d}


def exact(case, seed):
    t = _inputs(case, seed)
    kind = case["kind"]
    if kind in ("loss", "train"):
        return _exact_cross_entropy(case, t)
    if kind in ("norm", "ntrain"):
        x = t["x"].double()
        mean = x.mean(1)
        var = x.var(1, unbiased=False)
        rstd = (var + EPS_NORM).rsqrt()
        w, b = t["weight"].double(), t["bias"].double()
        h = (x - mean[:, None]) * rstd[:, None]
        out = dict(y=torch.addcmul(b, h, w), mean=mean, rstd=rstd)
        if kind == "ntrain":
            dy = t["dy"].double()
            # The row's Jacobian (I - 1 1'/d - h h'/d) / sigma applied to dy w.
            a = dy * w
            a1, ah = a.sum(1) / case["d"], (a * h).sum(1) / case["d"]
            out["dx"] = (a - a1[:, None] - ah[:, None] * h) * rstd[:, None]
            out["dweight"] = (dy * h).sum(0)
            out["dbias"] = dy.sum(0)
        return out
    # Every piece begins at a multiple of BLOCK and the gaps between them do not
    # move: all pieces at once, the gaps put back.
    g, p = t["g"].double(), t["p"].double()
    m, v = t["m"].double(), t["v"].double()
    pieces, total = _pieces(case)
    at = torch.arange(total, device="cuda") // BLOCK
    if case["bits"] == 8:
        m, v = m * t["ms"].double()[at], (v * t["vs"].double()[at]) ** 2
    inside = torch.zeros(total, dtype=torch.bool, device="cuda")
    for a, length in pieces:
        inside[a:a + length] = True
    m1, v1 = m + (1.0 - BETA1) * (g - m), v + (1.0 - BETA2) * (g * g - v)
    by = m1 / ((v1 / (1.0 - BETA2 ** STEP)) ** 0.5 + EPS)
    p1 = p - LR * DECAY * p - LR / (1.0 - BETA1 ** STEP) * by
    out = dict(p=torch.where(inside, p1, p))
    if case["bits"] == 32:
        return dict(out, m=torch.where(inside, m1, m), v=torch.where(inside, v1, v))
    for a, code, scale in ((m1, "m", "ms"), (v1 ** 0.5, "v", "vs")):
        a = torch.where(inside, a, 0.0)
        top = torch.zeros(total // BLOCK, dtype=torch.float64, device="cuda")
        top.scatter_reduce_(0, at, a.abs(), "amax")
        out[scale] = top / TOP
        out[code] = torch.where(inside, a / out[scale][at].clamp(min=1e-300),
                                t[code].double())  # what the codes round
    return out


def _exact_cross_entropy(case, t):
    x, w, labels = t["x"].double(), t["w"].double(), t["labels"].long()
    n, k = case["n"], case["k"]
    counted = max(1, int((labels >= 0).sum()))
    losses, lses, dx = [], [], []
    dw = torch.zeros_like(w)
    rows = max(1, (1 << 28) // k)
    for a in range(0, n, rows):
        xa, la = x[a:a + rows], labels[a:a + rows]
        z = xa @ w.t()
        lse = torch.logsumexp(z, 1)
        has = la >= 0
        r = torch.arange(z.shape[0], device="cuda")[has]
        loss = torch.zeros_like(lse)
        loss[has] = lse[has] - z[r, la[has]]
        losses.append(loss)
        lses.append(lse)
        if case["kind"] == "train":
            g = z.sub_(lse[:, None]).exp_()
            g[r, la[has]] -= 1.0
            g[~has] = 0.0
            g.div_(counted)
            dx.append(g @ w)
            dw.addmm_(g.t(), xa)
    out = dict(loss=torch.cat(losses), lse=torch.cat(lses))
    if case["kind"] == "train":
        out.update(dx=torch.cat(dx), dw=dw)
    return out
