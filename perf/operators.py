"""What a transformer block's linear layers, norms and optimizer step cost, and what they return.

Three operators that a training step of a decoder block runs side by side:

* ``linear``: a matrix product whose epilogue adds the bias, applies the activation and adds the
  residual stream -- forward alone (serving, down to one token) or with its gradients;
* ``norm``: the norm after a block, its gate and residual scale, the residual add and the norm
  before the next block -- forward alone or with its gradients;
* ``adamw``: one AdamW step over every tensor of a model, with its moments in 32 or in 8 bits.

``run`` computes them from elementary torch operations in 32 bits, or, where ``own`` is true, with
the framework's calls; ``exact`` computes them in 64 bits.
"""
import itertools
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5  # of the norms
BETAS, ADAM_EPS, LR, WEIGHT_DECAY, CLIP = (0.9, 0.95), 1e-8, 1e-4, 0.1, 0.7
BLOCK = 256  # elements of one tensor that share the scale of an 8-bit moment
TOP = 448.0  # the largest value of float8_e4m3fn


# ------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of a decode step through a wide up projection: the weight's bytes alone
        _linear("linear-one-token", False, 1, 4096, 14336, "silu", "bf16", False, False),
        # a prompt of odd length through a layer whose widths are no multiples of a tile
        _linear("linear-ragged-fp16", False, 777, 1000, 2504, "gelu", "fp16", True, True),
        # the first linear of a feed-forward block, trained: bias and GELU in the epilogue
        _linear("linear-train-up", True, 8192, 1280, 5120, "gelu", "bf16", True, False),
        # a micro-batch of six 4096-token samples through the widest layer, residual added
        _linear("linear-train-wide", True, 24576, 4096, 14336, "gelu_tanh", "bf16", True, True),
        # eight sequences decoding one token each: norm after the block, gate, add, norm before the next
        _norm("norm-decode", False, 8, 4096, "rms", True, "channel", True, False, "bf16"),
        # pre-norm blocks with LayerNorm: residual add and norm, trained
        _norm("norm-train-layer", True, 16384, 1280, "layer", False, "none", True, True, "bf16"),
        # an odd width in 32 bits, both norms and a scalar gate, trained
        _norm("norm-train-odd-fp32", True, 3001, 1001, "layer", True, "scalar", True, True, "fp32"),
        # a micro-batch of six 4096-token samples, sandwich norms with a channel gate, trained
        _norm("norm-train-sandwich", True, 24576, 4096, "rms", True, "channel", True, False, "bf16"),
        # a toy model's step: many small tensors, latency counts
        _adamw("adamw-toy-32", 48, 3, 65, 32, False, "fp32"),
        # a small model, fp32 master weights over bf16 ones, moments in 8 bits
        _adamw("adamw-small-8", 512, 8, 50257, 8, True, "bf16"),
        # a model trained in 32 bits throughout, as under autocast
        _adamw("adamw-medium-32", 1280, 12, 50257, 32, False, "fp32"),
        # a larger model with 8-bit moments, fp32 gradients accumulated over micro-batches
        _adamw("adamw-large-8", 2048, 12, 50304, 8, True, "fp32"),
    ]


def _linear(name, train, rows, inner, cols, act, dtype, bias, residual):
    return {"name": name, "op": "linear", "train": train, "rows": rows, "inner": inner, "cols": cols, "act": act,
            "dtype": dtype, "bias": bias, "residual": residual}


def _norm(name, train, rows, width, kind, post, gate, residual, bias, dtype):
    return {"name": name, "op": "norm", "train": train, "rows": rows, "width": width, "kind": kind, "post": post,
            "gate": gate, "residual": residual, "bias": bias, "dtype": dtype}


def _adamw(name, width, layers, vocab, bits, master, grad):
    return {"name": name, "op": "adamw", "width": width, "layers": layers, "vocab": vocab, "bits": bits,
            "master": master, "grad": grad}


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "norm", "adamw"))
    if op == "linear":
        inner, cols = (_spread(rng, 33, 8192) // k * k or k for k in (rng.choice((1, 8, 64)), rng.choice((1, 8, 64))))
        train = rng.random() < 0.6
        case = _linear("", train, _spread(rng, 1, 16384), inner, cols,
                       rng.choice(("none", "relu", "gelu", "gelu_tanh", "silu")), rng.choice(("bf16", "bf16", "fp16")),
                       rng.random() < 0.7, rng.random() < 0.5)
    elif op == "norm":
        post, dtype = rng.random() < 0.6, rng.choice(("bf16", "bf16", "fp16", "fp32"))
        width = _spread(rng, 16, 8192)
        width = width if rng.random() < 0.4 else max(8, width // 8 * 8)
        case = _norm("", rng.random() < 0.7, min(_spread(rng, 1, 24576), (1 << (25 if dtype == "fp32" else 26)) // width), width,
                     rng.choice(("rms", "layer")), post,
                     rng.choice(("none", "scalar", "channel")), post or rng.random() < 0.8, rng.random() < 0.5, dtype)
        if case["kind"] == "rms":
            case["bias"] = False
        if not case["residual"]:
            case["gate"] = "none"
    else:
        width = _spread(rng, 16, 1536)
        case = _adamw("", width, _spread(rng, 2, 24 if width < 1024 else 8), _spread(rng, 65, 50304),
                      rng.choice((8, 32)), rng.random() < 0.5, rng.choice(("bf16", "fp32")))
        if not case["master"]:
            case["grad"] = "fp32"
    del case["name"]
    return case


# ----------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    return {"linear": _prepare_linear, "norm": _prepare_norm, "adamw": _prepare_adamw}[case["op"]](case, gen)


def _randn(gen, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std).to(dtype)


def _leaf(t, train):
    return t.requires_grad_(True) if train else t


def _prepare_linear(c, gen):
    t, train, m, k, n = DTYPES[c["dtype"]], c["train"], c["rows"], c["inner"], c["cols"]
    return {
        "op": "linear", "act": c["act"], "train": train,
        "x": _leaf(_randn(gen, m, k, dtype=t), train),
        "w": _leaf(_randn(gen, n, k, std=k ** -0.5, dtype=t), train),
        "b": _leaf(_randn(gen, n, std=0.1, dtype=t), train) if c["bias"] else None,
        "r": _leaf(_randn(gen, m, n, dtype=t), train) if c["residual"] else None,
        "dy": _randn(gen, m, n, std=0.05, dtype=t) if train else None,
    }


def _prepare_norm(c, gen):
    t, train, m, d = DTYPES[c["dtype"]], c["train"], c["rows"], c["width"]

    def weight(around):
        return _leaf((around + _randn(gen, d, std=0.1)).to(t), train)

    gate = {"none": 0, "scalar": 1, "channel": d}[c["gate"]]
    return {
        "op": "norm", "kind": c["kind"], "train": train, "scale": 0.5 if c["post"] else 1.0,
        "h": _leaf(_randn(gen, m, d, std=0.7, dtype=t), train),
        "r": _leaf(_randn(gen, m, d, std=2.0, dtype=t), train) if c["residual"] else None,
        "gate": _leaf(_randn(gen, gate, std=0.3, dtype=t), train) if gate else None,
        "post_w": weight(1.0) if c["post"] else None,
        "post_b": weight(0.0) if c["post"] and c["bias"] else None,
        "pre_w": weight(1.0),
        "pre_b": weight(0.0) if c["bias"] else None,
        "dy": _randn(gen, m, d, std=0.05, dtype=t) if train else None,
        "ds": _randn(gen, m, d, std=0.05, dtype=t) if train else None,
    }


def _shapes(c):
    """The tensors of a decoder model: (shape, whether it decays), in the order that a program has them."""
    d = c["width"]
    got = [((c["vocab"], d), True), ((1024, d), True)]
    layer = [((d,), False), ((d,), False), ((3 * d, d), True), ((3 * d,), False), ((d, d), True), ((d,), False),
             ((d,), False), ((d,), False), ((4 * d, d), True), ((4 * d,), False), ((d, 4 * d), True), ((d,), False)]
    return got + layer * c["layers"] + [((d,), False), ((d,), False)]


def _first8(x):
    """A moment in 8 bits, rounded to nearest, and the scales of its blocks."""
    x = x.view(-1, BLOCK)
    scale = x.abs().amax(1, keepdim=True) / TOP
    return (x / scale.clamp_min(1e-30)).clamp_(-TOP, TOP).to(torch.float8_e4m3fn).view(-1), scale


def _prepare_adamw(c, gen):
    shapes = _shapes(c)
    sizes = [math.prod(s) for s, _ in shapes]
    blocks = [-(-n // BLOCK) for n in sizes]
    total = sum(blocks) * BLOCK  # every tensor lies at the start of a block of one allocation
    ends = [0, *itertools.accumulate(blocks)]
    at = [e * BLOCK for e in ends[:-1]]
    start, size = (torch.tensor(v, device="cuda").repeat_interleave(torch.tensor(blocks, device="cuda") * BLOCK)
                   for v in (at, sizes))
    real = torch.arange(total, device="cuda") - start < size
    del start, size
    master = _randn(gen, total, std=0.02).mul_(real)
    s = {"op": "adamw", "bits": c["bits"], "blocks": blocks, "step": 37,
         "wd": [WEIGHT_DECAY if decays else 0.0 for _, decays in shapes],
         "clip": torch.full((1,), CLIP, device="cuda"),
         "grad": (_randn(gen, total, std=1e-3).mul_(real)).to(DTYPES[c["grad"]]),
         "master": master if c["master"] else None, "param": master.bfloat16() if c["master"] else master}
    m, v = _randn(gen, total, std=3e-4).mul_(real), _randn(gen, total, std=1e-3).square_().mul_(real)
    if c["bits"] == 8:
        (s["exp_avg"], m), (s["exp_avg_sq"], v) = _first8(m), _first8(v.sqrt_())
        s["scales"] = torch.cat((m, v), 1)
    else:
        s["exp_avg"], s["exp_avg_sq"], s["scales"] = m, v, None

    def views(flat):
        return None if flat is None else [flat[a: a + n].view(sh) for a, n, (sh, _) in zip(at, sizes, shapes)]

    s["lists"] = {k: views(s[k]) for k in ("param", "grad", "master", "exp_avg", "exp_avg_sq")}
    s["lists"]["scales"] = None if s["scales"] is None else [s["scales"][e: e + b] for e, b in zip(ends, blocks)]
    return s


# -------------------------------------------------------------------------------------------- run
def run(s):
    return {"linear": _run_linear, "norm": _run_norm, "adamw": _run_adamw}[s["op"]](s)


def _some(*ts):
    return [t for t in ts if t is not None]


def _run_linear(s):
    x, w, b, r, dy = s["x"], s["w"], s["b"], s["r"], s["dy"]
    if own:
        from scaletorch_amd import ops

        y = ops.linear_act(x, w, b, r, activation=s["act"])
        return [y, *torch.autograd.grad(y, _some(x, w, b, r), dy)] if s["train"] else [y]
    t = x.dtype
    with torch.no_grad():
        xf, wf = x.float(), w.float()
        z = xf @ wf.t()
        if b is not None:
            z += b.float()
        a, slope = _activation(z, s["act"], s["train"])
        y = (a if r is None else a + r.float()).to(t)
        if not s["train"]:
            return [y]
        dz = dy.float() * slope if slope is not None else dy.float()
        got = [y, (dz @ wf).to(t), (dz.t() @ xf).to(t)]
        if b is not None:
            got.append(dz.sum(0).to(t))
        return got if r is None else [*got, dy]


def _activation(z, kind, train):
    """The activation of z and, for training, its derivative (None: one)."""
    if kind == "none":
        return z, None
    if kind == "relu":
        return z.clamp_min(0), (z > 0).float() if train else None
    if kind == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p * (1 + z * (1 - p)) if train else None
    if kind == "gelu":
        p = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * p, p + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi)) if train else None
    c = math.sqrt(2 / math.pi)
    p = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1 + p), (0.5 * (1 + p) + 0.5 * z * (1 - p * p) * c * (1 + 3 * 0.044715 * z * z)) if train else None


def _run_norm(s):
    h, r, gate, pw, pb, nw, nb = (s[k] for k in ("h", "r", "gate", "post_w", "post_b", "pre_w", "pre_b"))
    if own:
        from scaletorch_amd import ops

        y, out = ops.block_norm(h, r, kind=s["kind"], post_weight=pw, post_bias=pb, gate=gate, scale=s["scale"],
                                pre_weight=nw, pre_bias=nb, eps=EPS)
        if not s["train"]:
            return [y, out]
        return [y, out, *torch.autograd.grad((y, out), _some(h, r, gate, pw, pb, nw, nb), (s["dy"], s["ds"]))]
    t, scale = h.dtype, s["scale"]
    with torch.no_grad():
        hf = u = h.float()
        hhat = rstd = None
        if pw is not None:
            hhat, rstd = _normalize(hf, s["kind"])
            u = hhat * pw.float()
            if pb is not None:
                u = u + pb.float()
        v = u * scale if gate is None else u * (gate.float() * scale)
        out = v if r is None else r.float() + v
        ohat, orstd = _normalize(out, s["kind"])
        y = ohat * nw.float()
        if nb is not None:
            y = y + nb.float()
        if not s["train"]:
            return [y.to(t), out.to(t)]
        dy = s["dy"].float()
        dout = _normalize_back(dy * nw.float(), ohat, orstd, s["kind"]) + s["ds"].float()
        dv = dout * scale
        du = dv if gate is None else dv * gate.float()
        dh = du if pw is None else _normalize_back(du * pw.float(), hhat, rstd, s["kind"])
        dgate = None if gate is None else ((dv * u).sum(0) if gate.numel() > 1 else (dv * u).sum().view(1))
        grads = [dh, None if r is None else dout, dgate, None if pw is None else (du * hhat).sum(0),
                 None if pb is None else du.sum(0), (dy * ohat).sum(0), None if nb is None else dy.sum(0)]
        return [y.to(t), out.to(t), *(g.to(t) for g in grads if g is not None)]


def _normalize(x, kind):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * rstd, rstd


def _normalize_back(g, xhat, rstd, kind):
    got = g - xhat * (g * xhat).mean(-1, keepdim=True)
    if kind == "layer":
        got = got - g.mean(-1, keepdim=True)
    return got * rstd


def _run_adamw(s):
    if own:
        from scaletorch_amd import ops

        a = s["lists"]
        ops.adamw_multi_(a["param"], a["grad"], a["exp_avg"], a["exp_avg_sq"], step=s["step"], lr=LR, betas=BETAS,
                         eps=ADAM_EPS, weight_decay=s["wd"], masters=a["master"], scales=a["scales"],
                         clip_coef=s["clip"], scale_grads=s["grad"].dtype == torch.float32)  # fp32 ones stay clipped
        return _adamw_state(s)
    (b1, b2), t = BETAS, s["step"]
    p = s["param"] if s["master"] is None else s["master"]
    g = s["grad"].float().mul_(s["clip"])
    m, r = s["exp_avg"].float().view(-1, BLOCK), s["exp_avg_sq"].float().view(-1, BLOCK)
    if s["bits"] == 8:
        m = m * s["scales"][:, :1]
        r = (r * s["scales"][:, 1:]).square_()
    g = g.view(-1, BLOCK)
    m = m * b1 + g * (1 - b1)
    v = r * b2 + (g * g) * (1 - b2)
    root = v.sqrt()
    upd = (m * (1 / (1 - b1 ** t))) / (root * (1 / math.sqrt(1 - b2 ** t)) + ADAM_EPS)
    wd = torch.tensor([1 - LR * w for w in s["wd"]], device=p.device)
    keep = torch.repeat_interleave(wd, torch.tensor(s["blocks"], device=p.device), output_size=sum(s["blocks"]))
    p.copy_((p.view(-1, BLOCK) * keep[:, None] - upd * LR).view(-1))
    if s["master"] is not None:
        s["param"].copy_(p)
    if s["bits"] == 32:
        s["exp_avg"].copy_(m.view(-1))
        s["exp_avg_sq"].copy_(v.view(-1))
        return _adamw_state(s)
    low, high = _offsets(m.numel(), t, m.device)
    _store8(s, 0, "exp_avg", m, low)
    _store8(s, 1, "exp_avg_sq", root, high)
    return _adamw_state(s)


def _adamw_state(s):
    return {k: s[k] for k in ("param", "master", "exp_avg", "exp_avg_sq", "scales") if s[k] is not None}


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _offsets(n, step, device):
    """The 16 random bits with which each element of the step rounds its two moments: hashes of its place in the blocks."""
    key = _mix((step * 0x9E3779B9) & 0xFFFFFFFF)
    i = torch.arange(n, dtype=torch.int64, device=device)
    h = _mix((i & 0xFFFFFFFF) ^ _mix((i >> 32) ^ key))
    return h & 0xFFFF, h >> 16


def _store8(s, k, name, x, r16):
    """Blocks x in 8 bits: scaled so that the largest value is the type's largest, the others rounded up or down with r16."""
    top = x.abs().amax(1, keepdim=True)
    s["scales"][:, k: k + 1] = top * (1 / TOP)
    a = (x.abs() * torch.where(top > 2.0 ** -100, TOP / top, 0.0)).clamp_max_(TOP)
    tiny = torch.where(a < 2.0 ** -6, 2.0 ** -6, 0.0)  # below it the steps are equal: those of the binade above
    bits = (a + tiny).view(torch.int32).to(torch.int64) + (r16.view_as(a) << 4)
    q = (bits & ~0xFFFFF).to(torch.int32).view(torch.float32) - tiny
    if k:
        q = torch.where(a > 0, q.clamp_min(2.0 ** -9), q)  # a root that is not zero stays so
    s[name].copy_(torch.copysign(q, x).to(torch.float8_e4m3fn).view(-1))


# ------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "linear":
        m, k, n, e = c["rows"], c["inner"], c["cols"], 2
        read = m * k + n * k + n * c["bias"] + m * n * c["residual"]
        if not c["train"]:
            return {"bytes": e * (read + m * n), "flops": 2 * m * n * k}
        return {"bytes": e * (2 * read - m * n * c["residual"] + 2 * m * n), "flops": 6 * m * n * k}
    if c["op"] == "norm":
        e, md = (4 if c["dtype"] == "fp32" else 2), c["rows"] * c["width"]
        streams = 3 + c["residual"]  # h, the residual, y and the new stream
        if c["train"]:
            streams += 3 + c["residual"]  # dy, ds, dh and the residual's gradient
        return {"bytes": e * streams * md, "flops": (30 if c["train"] else 12) * md}
    n = sum(math.prod(s) for s, _ in _shapes(c))
    per = (DTYPES[c["grad"]].itemsize + 8 + (2 if c["master"] else 0)
           + (4 if c["bits"] == 8 else 16))  # read and write; the scales are a 64th of a byte each
    return {"bytes": per * n, "flops": 16 * n}


# ------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "norm": _exact_norm, "adamw": _exact_adamw}[case["op"]](s)


def _double(t, train):
    return None if t is None else t.detach().double().requires_grad_(train)


def _exact_linear(s):
    x, w, b, r = (_double(s[k], s["train"]) for k in ("x", "w", "b", "r"))
    z = x.mm(w.t()) if b is None else torch.addmm(b, x, w.t())
    if s["act"] == "relu":
        z = torch.relu(z)
    elif s["act"] == "silu":
        z = z * torch.sigmoid(z)
    elif s["act"] == "gelu":
        z = z * torch.erfc(-z / math.sqrt(2.0)) / 2
    elif s["act"] == "gelu_tanh":
        z = z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))  # (1 + tanh(a)) / 2 = sigmoid(2 a)
    y = z if r is None else z + r
    if not s["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, _some(x, w, b, r), s["dy"].double())]


def _exact_norm(s):
    h, r, gate, pw, pb, nw, nb = (_double(s[k], s["train"]) for k in ("h", "r", "gate", "post_w", "post_b", "pre_w", "pre_b"))

    def norm(x, w, b):
        if s["kind"] == "rms":
            return x * w / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
        got = (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + EPS).sqrt() * w
        return got if b is None else got + b

    u = h if pw is None else norm(h, pw, pb)
    out = s["scale"] * u * (1.0 if gate is None else gate) + (0.0 if r is None else r)
    y = norm(out, nw, nb)
    if not s["train"]:
        return [y, out]
    grads = torch.autograd.grad((y, out), _some(h, r, gate, pw, pb, nw, nb), (s["dy"].double(), s["ds"].double()))
    return [y.detach(), out.detach(), *grads]


def _exact_adamw(s):
    (b1, b2), t, eight = BETAS, s["step"], s["bits"] == 8
    p = (s["param"] if s["master"] is None else s["master"]).double()
    g = s["grad"].double() * s["clip"].double()
    m, v = s["exp_avg"].double(), s["exp_avg_sq"].double()
    if eight:
        sc = s["scales"].double()
        m, v = m * sc[:, 0].repeat_interleave(BLOCK), (v * sc[:, 1].repeat_interleave(BLOCK)) ** 2
    m.mul_(b1).add_(g, alpha=1 - b1)
    v.mul_(b2).addcmul_(g, g, value=1 - b2)
    del g
    wd = torch.tensor(s["wd"], device=p.device, dtype=torch.float64)
    wd = wd.repeat_interleave(torch.tensor(s["blocks"], device=p.device) * BLOCK)
    p.sub_(p * wd, alpha=LR).addcdiv_(m / (1 - b1 ** t), (v / (1 - b2 ** t)).sqrt() + ADAM_EPS, value=-LR)
    got = {"param": p, "exp_avg": m, "exp_avg_sq": v}
    if s["master"] is not None:
        got["master"] = p
    if eight:
        low, high = _offsets(m.numel(), t, m.device)
        a, b = _exact8(m, low, 0.0), _exact8(v.sqrt_(), high, 2.0 ** -9)
        got |= {"exp_avg": a[0], "exp_avg_sq": b[0], "scales": torch.stack((a[1], b[1]), 1)}
    return got


def _exact8(x, r16, least):
    x = x.view(-1, BLOCK)
    top = x.abs().amax(1, keepdim=True)
    a = torch.where(top > 0, x.abs() * TOP / top, 0.0)
    step = torch.exp2(torch.frexp(a).exponent.clamp_min(-5).double() - 4)  # four significant bits, 2^-9 at least
    q = ((a / step + r16.view_as(a).double() / 65536).floor() * step).clamp_max(TOP)
    q = torch.where(a > 0, q.clamp_min(least), q)
    return (q * x.sign()).view(-1), (top / TOP).view(-1)
