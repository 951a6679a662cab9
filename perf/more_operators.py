"""The operators of a classifier that answers in 8 bits and is tuned by what its
answers were worth, as measured cases.

One case is a dict; its "kind" says which operator runs:

  norm8   HipDevice.rms_norm of rows and what is added to them, into 8-bit codes with a scale
          for every 128 columns
  ntrain  the same into rows of the case's type, then HipDevice.rms_norm_grad: the gradients
          of the rows and of the weight
  product HipDevice.product8: rows in 8 bits times classes in 8 bits, the logits
  answer  HipDevice.log_probs: log probabilities of given classes, entropies and the likeliest
          classes of rows of logits
  policy  HipDevice.log_probs, then HipDevice.log_probs_grad: the gradient of the logits
  clip    GradNorm.clip over a list of tensors: their norm, and the gradients brought to it

Inputs and outputs have the case's "type"; 8-bit values are float8_e4m3fn codes with float32
scales; statistics, log probabilities and norms are float32.
"""

import math

import torch

own = False

NONE = -1          # a row without a given class (0xFFFFFFFF), a place without an alternative
BLOCK = 128        # columns (of classes: and rows) that share a scale
TOP = 448.0        # the largest float8_e4m3fn
EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_DEV = []


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # One row on its way to the classes: latency.
        dict(name="norm8_1x1024_bf16", kind="norm8", n=1, d=1024, type="bf16"),
        # Odd rows in half precision, whose last block of columns is a short one.
        dict(name="norm8_10007x300_f16", kind="norm8", n=10007, d=300, type="f16"),
        # One training batch of the headline clustering's rows.
        dict(name="ntrain_16384x768_bf16", kind="ntrain", n=16384, d=768, type="bf16"),
        # One row against a large codebook: reading the classes once.
        dict(name="product_1x1024_k16384_bf16", kind="product", n=1, d=1024, k=16384,
             type="bf16"),
        # Odd sizes everywhere, exact logits.
        dict(name="product_10007x300_k1000_f32", kind="product", n=10007, d=300, k=1000,
             type="f32"),
        # The headline batch against its clusters.
        dict(name="product_16384x768_k1024_bf16", kind="product", n=16384, d=768, k=1024,
             type="bf16"),
        # A large vocabulary, one class short of a round number.
        dict(name="product_8192x1024_k131071_bf16", kind="product", n=8192, d=1024, k=131071,
             type="bf16"),
        # One row's answer from that vocabulary: latency over a long row.
        dict(name="answer_1_k131071_bf16", kind="answer", n=1, k=131071, top=8, type="bf16"),
        # Many short rows of odd length.
        dict(name="answer_10007_k1000_f32", kind="answer", n=10007, k=1000, top=5, type="f32"),
        # A tuning step on half a batch of answers from the large vocabulary.
        dict(name="policy_4096_k131071_bf16", kind="policy", n=4096, k=131071, type="bf16"),
        # The gradients of a small head: its classes and the norm before it.
        dict(name="clip_256x384_f32", kind="clip", k=256, d=384, layers=1, type="f32"),
        # The large vocabulary's, and two dozen small tensors that begin anywhere.
        dict(name="clip_131071x1001_bf16", kind="clip", k=131071, d=1001, layers=24,
             type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _dim(rng):
    """Mostly the widths that embeddings have, one in four any width."""
    if rng.random() < 0.25:
        return rng.randint(16, 1100)
    return rng.choice([64, 96, 100, 128, 200, 256, 300, 384, 512, 640, 768, 1024])


def draw(rng):
    kind = rng.choice(["norm8", "ntrain", "product", "product", "answer", "policy", "clip"])
    type_ = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind in ("norm8", "ntrain"):
        return dict(kind=kind, n=_log(rng, 1, 100_000), d=_dim(rng), type=type_)
    if kind == "clip":
        return dict(kind=kind, k=_log(rng, 16, 32_768), d=_dim(rng), layers=rng.randint(1, 24),
                    type=type_)
    n, k, d = _log(rng, 1, 16_384), _log(rng, 16, 131_071), _dim(rng)
    each, most = (d, 1 << 40) if kind == "product" else (1, 1 << 29)
    while n * k * each * (2 if type_ == "f32" else 1) > most:
        n, k = (n + 1) // 2, (k + 1) // 2
    if kind == "product":
        return dict(kind=kind, n=n, d=d, k=k, type=type_)
    if kind == "answer":
        return dict(kind=kind, n=n, k=k, top=rng.randint(1, min(16, k)), type=type_)
    return dict(kind=kind, n=n, k=k, type=type_)


# ----------------------------------------------------------------- the inputs
def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(1_000_003 * int(seed) + salt)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _blocks(length):
    return -(-length // BLOCK)


def _wide(d):
    """Bytes of a row of d codes: rows begin at multiples of 16."""
    return -(-d // 16) * 16


def _coded(a, rows):
    """a in 8 bits, every rows x BLOCK of it with the scale largest / TOP."""
    n, d = a.shape
    full = torch.nn.functional.pad(a, (0, _blocks(d) * BLOCK - d, 0, -n % rows))
    tiles = full.view(-1, rows, _blocks(d), BLOCK)
    scale = tiles.abs().amax((1, 3)) / TOP
    q = tiles / torch.where(scale > 0, scale, torch.ones_like(scale))[:, None, :, None]
    q = q.clamp_(-TOP, TOP).to(torch.float8_e4m3fn).view(full.shape)
    return q[:n, :_wide(d)].contiguous(), scale


def _loss_scale(case):
    """Gradients in half precision are those of so many times the loss."""
    return 1024.0 if case["type"] == "f16" else 1.0


def _inputs(case, seed):
    """The case's tensors, from the seed alone."""
    kind, type_ = case["kind"], TYPES[case["type"]]
    g = _gen(seed, 2)
    if kind in ("norm8", "ntrain"):
        n, d = case["n"], case["d"]
        # Rows of sizes of their own, a few columns larger than the others, and what a layer
        # adds to them.
        column = 1.0 + 7.0 * (_rand(g, d) < 0.02).float()
        x = _randn(g, n, d).mul_(0.5 + 2.0 * _rand(g, n, 1)).mul_(column)
        t = dict(x=x.to(type_), r=_randn(g, n, d).mul_(0.3).to(type_),
                 weight=_randn(g, d).mul_(0.1).add_(1.0).to(type_))
        if kind == "ntrain":
            t["dy"] = _randn(g, n, d).mul_(_loss_scale(case) / n).to(type_)
            t["dh"] = _randn(g, n, d).mul_(_loss_scale(case) / n).to(type_)
        return t
    if kind == "product":
        n, d, k = case["n"], case["d"], case["k"]
        # A codebook's rows, and rows after a norm that are part noise and part their class.
        w = _randn(g, k, d).div_(math.sqrt(d))
        at = torch.randint(k, (n,), generator=g, device="cuda")
        x = _randn(g, n, d).add_(w[at] * 8.0 * _rand(g, n, 1))
        t = {}
        t["x"], t["xs"] = _coded(x, 1)
        t["w"], t["ws"] = _coded(w, BLOCK)
        return t
    if kind in ("answer", "policy"):
        n, k = case["n"], case["k"]
        # Logits of which one stands out to some degree; three rows in four have classes that
        # may not be answered, one in 500 none that may; the given class is the one that
        # stands out, another or none.
        z = _randn(g, n, k).mul_(2.0)
        best = torch.randint(k, (n, 1), generator=g, device="cuda")
        z.scatter_add_(1, best, 16.0 * _rand(g, n, 1))
        share = 0.5 * (_rand(g, n, 1) - 0.25).clamp_(min=0.0)
        share[_rand(g, n, 1) < 0.002] = 1.0
        z.masked_fill_(_rand(g, n, k) < share, -math.inf)
        other = torch.randint(k, (n,), generator=g, device="cuda")
        tokens = torch.where(_rand(g, n) < 0.7, best[:, 0], other)
        tokens[_rand(g, n) < 0.02] = NONE
        t = dict(z=z.to(type_), tokens=tokens.to(torch.int32))
        if kind == "policy":
            # What the answers were worth beside the mean, and a small weight on entropy.
            t["glogp"] = _randn(g, n).mul_(_loss_scale(case) / n)
            t["gentropy"] = _rand(g, n).mul_(0.01 * _loss_scale(case) / n)
        return t
    # The tensors lie one behind the other in one buffer, as a program keeps them that
    # reduces them at once. Most steps have a norm to bring down.
    total = sum(_lengths(case))
    return dict(g=_randn(g, total).mul_(0.02).to(type_),
                max_norm=0.02 * math.sqrt(total) * (0.25 + (seed % 8) / 8))


def _lengths(case):
    return [case["k"] * case["d"]] + [case["d"]] * (2 * case["layers"])


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
    dev, kind = _DEV[0], case["kind"]
    kinds = {torch.float32: E.F32, torch.int32: E.U32, torch.float16: E.F16,
             torch.bfloat16: E.BF16, torch.float8_e4m3fn: E.F8}
    wrap = lambda v: dev.wrap(v.data_ptr(), v.numel(), kinds[v.dtype])  # noqa: E731
    f = lambda *shape: torch.zeros(*shape, device="cuda")  # noqa: E731
    if kind == "clip":
        out = dict(state=f(2), g=torch.zeros_like(t["g"]))
        at, grads, outs = 0, [], []
        for length in _lengths(case):
            grads.append(wrap(t["g"][at:at + length]))
            outs.append(wrap(out["g"][at:at + length]))
            at += length
        return dict(plan=E.GradNorm(dev, grads, outs), out=dict(norm=out["state"][:1], g=out["g"]),
                    b_state=wrap(out["state"]))
    n = case["n"]
    if kind in ("norm8", "ntrain"):
        d = case["d"]
        out = dict(h=torch.zeros_like(t["x"]))
        if kind == "norm8":
            out.update(y=torch.zeros(n, _wide(d), device="cuda").to(torch.float8_e4m3fn),
                       scales=f(n, _blocks(d)))
        else:
            out.update(y=torch.zeros_like(t["x"]), rstd=f(n), dx=torch.zeros_like(t["x"]),
                       dweight=f(d))
    elif kind == "product":
        out = dict(y=torch.zeros(n, case["k"], dtype=TYPES[case["type"]], device="cuda"))
    else:
        out = dict(logp=f(n), lse=f(n), entropy=f(n))
        if kind == "answer":
            out.update(ids=torch.zeros(n, case["top"], dtype=torch.int32, device="cuda"),
                       top=f(n, case["top"]))
        else:
            out.update(dz=torch.zeros_like(t["z"]))
    o = dict(dev=dev, out=dict(out), **{"b_" + k: wrap(v) for k, v in {**t, **out}.items()})
    if kind == "norm8":
        o["out"]["y"] = out["y"][:, :case["d"]]
    return o


# ---------------------------------------------------------------- the one pass
def run(s):
    return _run_own(s["case"], s["t"], s["own"]) if own else _PLAIN[s["case"]["kind"]](
        s["case"], s["t"])


def _run_own(case, t, o):
    kind = case["kind"]
    if kind == "clip":
        o["plan"].clip(o["b_state"], t["max_norm"])
        return o["out"]
    dev, n = o["dev"], case["n"]
    if kind == "norm8":
        dev.rms_norm(o["b_x"], n, case["d"], o["b_weight"], o["b_y"], residual=o["b_r"],
                     h=o["b_h"], scales=o["b_scales"], eps=EPS)
    elif kind == "ntrain":
        dev.rms_norm(o["b_x"], n, case["d"], o["b_weight"], o["b_y"], residual=o["b_r"],
                     h=o["b_h"], rstd=o["b_rstd"], eps=EPS)
        dev.rms_norm_grad(o["b_dy"], o["b_h"], n, case["d"], o["b_weight"], o["b_rstd"],
                          o["b_dx"], o["b_dweight"], dh=o["b_dh"])
    elif kind == "product":
        dev.product8(o["b_x"], o["b_xs"], n, case["d"], o["b_w"], o["b_ws"], case["k"], o["b_y"])
    elif kind == "answer":
        dev.log_probs(o["b_z"], n, case["k"], o["b_tokens"], o["b_logp"], o["b_lse"],
                      entropy=o["b_entropy"], top=case["top"], top_ids=o["b_ids"],
                      top_logp=o["b_top"])
    else:
        dev.log_probs(o["b_z"], n, case["k"], o["b_tokens"], o["b_logp"], o["b_lse"],
                      entropy=o["b_entropy"])
        dev.log_probs_grad(o["b_z"], n, case["k"], o["b_tokens"], o["b_lse"], o["b_dz"],
                           entropy=o["b_entropy"], glogp=o["b_glogp"],
                           gentropy=o["b_gentropy"])
    return o["out"]


def _rms_norm(t):
    # The sum is kept in the rows' type, and the norm is of what is kept.
    h = (t["x"].float() + t["r"].float()).to(t["x"].dtype)
    rstd = 1.0 / (h.float().square().mean(1) + EPS).sqrt()
    return h, rstd, h.float() * rstd[:, None] * t["weight"].float()


def _plain_norm8(case, t):
    h, _, y = _rms_norm(t)
    q, scales = _coded(y, 1)
    return dict(h=h, y=q[:, :case["d"]], scales=scales)


def _plain_ntrain(case, t):
    h, rstd, y = _rms_norm(t)
    dy, hat = t["dy"].float(), h.float() * rstd[:, None]
    g = dy * t["weight"].float()
    dx = t["dh"].float() + rstd[:, None] * (g - hat * (g * hat).mean(1, keepdim=True))
    return dict(h=h, y=y.to(h.dtype), rstd=rstd, dx=dx.to(h.dtype), dweight=(dy * hat).sum(0))


def _plain_product(case, t):
    d, k = case["d"], case["k"]
    x = t["x"].float()[:, :d] * t["xs"].repeat_interleave(BLOCK, 1)[:, :d]
    ws = t["ws"].repeat_interleave(BLOCK, 0)[:k].repeat_interleave(BLOCK, 1)[:, :d]
    w = t["w"].float()[:, :d] * ws
    return dict(y=(x @ w.t()).to(TYPES[case["type"]]))


def _log_softmax(t):
    """lse, p and log p; a row without a class that may be answered has no p."""
    z = t["z"].float()
    top = z.amax(1, keepdim=True)
    lse = (z - top.clamp(min=-3e38)).exp().sum(1).log() + top[:, 0]
    lp = z - lse.clamp(min=-3e38)[:, None]
    p = lp.exp()
    return lse, p, lp


def _statistics(t):
    lse, p, lp = _log_softmax(t)
    entropy = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
    given = t["tokens"] >= 0
    logp = lp.gather(1, t["tokens"].long().clamp(min=0)[:, None])[:, 0]
    return dict(logp=torch.where(given, logp, torch.zeros_like(logp)), lse=lse,
                entropy=entropy), p, lp, given


def _plain_answer(case, t):
    out, _, lp, _ = _statistics(t)
    # The largest first, the lower class first among equals: values in an order of whole
    # numbers, with the class below them.
    z = (t["z"].float() + 0.0).view(torch.int32).long()
    z = torch.where(z < 0, -(z & 0x7FFFFFFF), z)
    key = z * 2 ** 32 + (2 ** 31 - torch.arange(case["k"], device="cuda"))
    ids = 2 ** 31 - (key.topk(case["top"], 1)[0] & 0xFFFFFFFF)
    top = lp.gather(1, ids)
    return dict(out, ids=torch.where(top == -math.inf, NONE, ids).to(torch.int32), top=top)


def _plain_policy(case, t):
    out, p, lp, given = _statistics(t)
    gl = torch.where(given, t["glogp"], torch.zeros_like(t["glogp"]))[:, None]
    plp = torch.where(p > 0, p * (lp + out["entropy"][:, None]), torch.zeros_like(p))
    dz = -gl * p - t["gentropy"][:, None] * plp
    some = (out["lse"] > -math.inf)[:, None]
    dz.scatter_add_(1, t["tokens"].long().clamp(min=0)[:, None],
                    torch.where(some, gl, torch.zeros_like(gl)))
    return dict(out, dz=dz.to(t["z"].dtype))


def _plain_clip(case, t):
    norm = t["g"].double().square().sum().sqrt()
    by = (t["max_norm"] / norm).clamp(max=1.0).float()
    return dict(norm=norm.float()[None], g=(t["g"].float() * by).to(t["g"].dtype))


_PLAIN = dict(norm8=_plain_norm8, ntrain=_plain_ntrain, product=_plain_product,
              answer=_plain_answer, policy=_plain_policy, clip=_plain_clip)


# ---------------------------------------------------- its size and its answer
def work(case):
    kind = case["kind"]
    e = 4 if case["type"] == "f32" else 2
    if kind == "clip":
        count = sum(_lengths(case))
        return {"bytes": 2 * count * e, "flops": 3 * count}
    n = case["n"]
    if kind == "norm8":
        d = case["d"]
        return {"bytes": n * d * (3 * e + 1) + 4 * n * _blocks(d) + d * e, "flops": 8 * n * d}
    if kind == "ntrain":
        # The backward pass is a call of its own and reads the sums again.
        d = case["d"]
        return {"bytes": 8 * n * d * e + 4 * n + d * (e + 4), "flops": 16 * n * d}
    k = case["k"]
    if kind == "product":
        d = case["d"]
        return {"bytes": (n + k) * d + n * k * e + 4 * (n + _blocks(k)) * _blocks(d),
                "flops": 2 * n * k * d}
    if kind == "answer":
        return {"bytes": n * k * e + n * (16 + 8 * case["top"]), "flops": 6 * n * k}
    # As above: the logits are read by both calls.
    return {"bytes": 3 * n * k * e + 24 * n, "flops": 14 * n * k}


def exact(case, seed):
    return _EXACT[case["kind"]](case, _inputs(case, seed))


def _exact_norm(case, t):
    h = (t["x"].double() + t["r"].double()).to(t["x"].dtype).double()
    d, w = case["d"], t["weight"].double()
    length = torch.linalg.vector_norm(h, dim=1, keepdim=True)
    sigma = torch.sqrt(length * length / d + EPS)
    unit = h / sigma
    y = unit * w
    if case["kind"] == "ntrain":
        # The row's Jacobian (I - u u'/d) / sigma applied to dy w.
        dy = t["dy"].double()
        a = dy * w
        dx = t["dh"].double() + (a - unit * ((a * unit).sum(1, keepdim=True) / d)) / sigma
        return dict(h=h, y=y, rstd=1.0 / sigma[:, 0], dx=dx, dweight=(dy * unit).sum(0))
    at = torch.arange(d, device="cuda") // BLOCK
    top = torch.zeros(case["n"], _blocks(d), dtype=torch.float64, device="cuda")
    top.scatter_reduce_(1, at.expand_as(y), y.abs(), "amax")
    scales = top / TOP
    return dict(h=h, y=y / scales[:, at].clamp(min=1e-300), scales=scales)  # what codes round


def _exact_product(case, t):
    n, d, k = case["n"], case["d"], case["k"]
    x, w = t["x"].double(), t["w"].double()
    xs, ws = t["xs"].double(), t["ws"].double()
    y = torch.zeros(n, k, dtype=torch.float64, device="cuda")
    for b in range(_blocks(d)):
        lo, hi = b * BLOCK, min(d, (b + 1) * BLOCK)
        by = ws[:, b].repeat_interleave(BLOCK)[:k, None]
        y.addmm_(x[:, lo:hi] * xs[:, b:b + 1], (w[:, lo:hi] * by).t())
    return dict(y=y)


def _exact_answers(case, t):
    n, k = case["n"], case["k"]
    tokens = t["tokens"].long()
    got = []
    rows = max(1, (1 << 27) // k)
    for a in range(0, n, rows):
        z, at = t["z"][a:a + rows].double(), tokens[a:a + rows]
        lse = torch.logsumexp(z, 1)
        some = lse > -math.inf
        lp = z - torch.where(some, lse, torch.zeros_like(lse))[:, None]
        p = torch.exp(lp)
        entropy = -torch.special.xlogy(p, p).sum(1)
        has = at >= 0
        r = torch.arange(z.shape[0], device="cuda")
        logp = torch.zeros_like(lse)
        logp[has] = lp[r[has], at[has]]
        one = dict(logp=logp, lse=lse, entropy=entropy)
        if case["kind"] == "answer":
            values, ids = torch.sort(lp, dim=1, descending=True, stable=True)
            one["top"] = values[:, :case["top"]].clone()
            one["ids"] = torch.where(one["top"] == -math.inf, NONE, ids[:, :case["top"]])
        else:
            gl = torch.where(has & some, t["glogp"][a:a + rows].double(), 0.0)
            ge = t["gentropy"][a:a + rows].double()
            # d logp / dz = onehot - p; d H / dz = -p (log p + H).
            dz = -gl[:, None] * p - ge[:, None] * (torch.special.xlogy(p, p) +
                                                   p * entropy[:, None])
            dz[r[has], at[has]] += gl[has]
            one["dz"] = dz
        got.append(one)
    return {name: torch.cat([one[name] for one in got]).to(
        torch.int32 if name == "ids" else torch.float64) for name in got[0]}


def _exact_clip(case, t):
    g = t["g"].double()
    norm = torch.linalg.vector_norm(g)
    return dict(norm=norm[None], g=g * min(1.0, t["max_norm"] / float(norm)))


_EXACT = dict(norm8=_exact_norm, ntrain=_exact_norm, product=_exact_product,
              answer=_exact_answers, policy=_exact_answers, clip=_exact_clip)
