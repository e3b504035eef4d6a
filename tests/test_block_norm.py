"""Norms around a gated residual (ops/block_norm.py, csrc/block_norm_*.hip) against 64 bits.

Tolerances.  The kernel computes in fp32 and rounds an output once, by at most u = eps / 2 of its
type relative to the value (one step of the smallest subnormal for fp16).  The fp32 sums over a row
of W columns are trees of depth log2 W per wave plus one addition a wave; 32 roundings of 2^-24 of
the row's largest terms bound s, y and the row gradients, here as an absolute term of the row's
scale.  The gradients of weights and gate are sums over R rows whose terms' magnitudes add up to M:
at most (R / 2 + 64) 2^-24 M for one worker's chain and the final additions.
"""
import pytest
import torch

from scaletorch_amd import ops
from scaletorch_amd.ops.block_norm import block_norm_ref

U32 = 2.0 ** -24
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
EPS = 1e-5
NAMES = ("h", "residual", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias")


def _inputs(device, rows, width, dtype, rdtype=None, wdtype=None, post=True, gate="channel", bias=True, residual=True,
            pre=True, seed=0, shift=0.0):
    g = torch.Generator().manual_seed(seed)

    def make(*shape, std=1.0, mean=0.0, dt=dtype):
        return (torch.randn(*shape, generator=g) * std + mean).to(dt).to(device)

    wdtype = wdtype or dtype
    c = dict(h=make(rows, width, mean=shift), residual=make(rows, width, std=2.0, mean=shift, dt=rdtype or dtype) if residual else None,
             gate={"none": None, "scalar": make(1, mean=0.5, dt=wdtype), "channel": make(width, std=0.5, dt=wdtype)}[gate],
             post_weight=make(width, std=0.2, mean=1, dt=wdtype) if post else None,
             post_bias=make(width, std=0.3, dt=wdtype) if post and bias else None,
             pre_weight=make(width, std=0.2, mean=1, dt=wdtype) if pre else None,
             pre_bias=make(width, std=0.3, dt=wdtype) if pre and bias else None)
    c["dy"] = make(rows, width)
    c["ds"] = make(rows, width, dt=rdtype or dtype)
    return c


def _run(c, kind, scale, use=("dy", "ds"), f=ops.block_norm):
    ts = {k: None if c[k] is None else c[k].detach().clone().requires_grad_(True) for k in NAMES}
    y, s = f(ts["h"], ts["residual"], kind=kind, scale=scale, eps=EPS, **{k: ts[k] for k in NAMES[2:]})
    outs = [(o, c[n]) for o, n in ((y, "dy"), (s, "ds")) if o is not None and n in use]
    some = [k for k in NAMES if ts[k] is not None]
    grads = torch.autograd.grad([o for o, _ in outs], [ts[k] for k in some], [g for _, g in outs], allow_unused=True)
    return y, s, dict(zip(some, grads))


def _ref(c, kind, scale, use=("dy", "ds")):
    d = {k: None if v is None else v.double() for k, v in c.items()}

    def f(h, residual, *, kind, scale, eps, post_weight, post_bias, gate, pre_weight, pre_bias):
        y, s = block_norm_ref(h, residual, kind == "layer", post_weight, post_bias, gate, scale, pre_weight, pre_bias, eps)
        return y, s

    return _run({k: None if v is None else v.cpu() for k, v in d.items()}, kind, scale, use, f)


def _close(got, ref, u, extra, what):
    """|got - ref| <= u |ref| (the rounding) + extra (absolute)."""
    got, ref = got.detach().double().cpu(), ref.detach().double()
    tiny = 2.0 ** -24 if got.dtype == torch.float16 else 0.0
    bad = (got - ref).abs() - (u * ref.abs() * 1.01 + extra + tiny + 2.0 ** -25)
    assert (bad <= 0).all(), f"{what}: {bad.max().item():.3g} past the bound at {ref.abs().max().item():.3g}"


def _compare(c, kind, scale, use=("dy", "ds")):
    y, s, g = _run(c, kind, scale, use)
    ry, rs, rg = _ref(c, kind, scale, use)
    u = torch.finfo(c["h"].dtype).eps / 2
    us = torch.finfo(s.dtype).eps / 2
    rows, width = c["h"].shape
    mag = lambda t: 0.0 if t is None else t.double().abs().max().item()  # noqa: E731
    big = {k: mag(c[k]) for k in c}
    wmax = max(1.0, big["pre_weight"]), max(1.0, big["post_weight"]) * max(1.0, big["gate"]) * abs(scale)
    # the smallest standard deviations of the rows, as eps leaves them, set how errors of x grow
    rstd2 = 1 / (rs.detach().var(-1, unbiased=False) + EPS).sqrt().min().item() if kind == "layer" else \
        1 / (rs.detach().pow(2).mean(-1) + EPS).sqrt().min().item()
    h64 = c["h"].double().cpu()
    rstd1 = 1.0 if c["post_weight"] is None else 1 / ((h64.var(-1, unbiased=False) if kind == "layer" else h64.pow(2).mean(-1)) + EPS).sqrt().min().item()
    smax = rs.detach().abs().max().item()
    # s: 32 roundings of the largest term in it, the normalised h included
    es = 32 * U32 * (smax + big["residual"] + wmax[1] * max(big["h"] * rstd1, 1.0) + big["post_bias"])
    _close(s, rs, us, es, "s")
    if y is not None:
        eyhat = 2 * es * rstd2 + 32 * U32 * max(1.0, smax * rstd2)
        _close(y, ry, u, wmax[0] * eyhat + 8 * U32 * (wmax[0] * smax * rstd2 + big["pre_bias"]), "y")
    eshat = 2 * es * rstd2 + 32 * U32 * max(1.0, smax * rstd2)
    gy = big["dy"] * wmax[0] if "dy" in use and y is not None else 0.0
    shat = max(1.0, smax * rstd2)
    eds = rstd2 * gy * (3 * eshat * shat + 64 * U32 * shat * shat) + 8 * U32 * big["ds"]
    dsmax = rg["residual"].abs().max().item() if "residual" in rg and rg["residual"] is not None else big["ds"] + rstd2 * gy * (1 + shat * shat)
    if "residual" in rg:
        _close(g["residual"], rg["residual"], us, eds, "dresidual")
    hhat = max(1.0, big["h"] * rstd1) if c["post_weight"] is not None else big["h"]
    edh = wmax[1] * (eds + 16 * U32 * dsmax) * rstd1 * (1 + hhat * hhat) + rstd1 * wmax[1] * dsmax * 128 * U32 * hhat * hhat
    _close(g["h"], rg["h"], u, edh, "dh")
    chain = (rows / 2 + 64) * U32
    sums = {"pre_weight": rows * big["dy"] * (eshat + chain * shat), "pre_bias": rows * big["dy"] * chain,
            "post_weight": rows * wmax[1] * (eds * hhat + dsmax * hhat * (chain + 32 * U32)),
            "post_bias": rows * wmax[1] * (eds + dsmax * chain),
            "gate": rows * abs(scale) * (max(1.0, big["post_weight"]) * hhat + big["post_bias"]) * (eds + dsmax * (chain + 32 * U32))}
    if c["gate"] is not None and c["gate"].numel() == 1:
        sums["gate"] *= width
    for k, e in sums.items():
        if k in rg:
            if rg[k] is None:
                assert g[k] is None or not g[k].any()
                continue
            _close(g[k], rg[k], torch.finfo(g[k].dtype).eps / 2, e, "d" + k)
    return y, s, g


SHAPES = [(1, 1), (3, 7), (5, 64), (9, 511), (4, 512), (6, 520), (130, 1000), (7, 1001), (33, 1280), (5, 4096),
          (3, 4099), (2, 8192), (2, 8191)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_all_parts(device, kind, rows, width, dtype):
    _compare(_inputs(device, rows, width, dtype), kind, 0.7)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", ["none", "scalar", "channel"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("pre", [False, True])
def test_each_part(device, kind, post, gate, bias, residual, pre):
    for k, (dtype, rdtype, wdtype) in enumerate(((torch.bfloat16, None, None), (torch.float16, torch.float32, torch.float32),
                                                 (torch.float32, None, None), (torch.bfloat16, torch.float32, None))):
        for scale in (1.0, 0.25):
            c = _inputs(device, 19, (264, 1001)[k % 2], dtype, rdtype if residual else None, wdtype, post, gate, bias,
                        residual, pre, seed=k)
            if not residual:
                c["ds"] = c["ds"].to(dtype)
            _compare(c, kind, scale)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("use", [("dy",), ("ds",)])
@pytest.mark.parametrize("post", [False, True])
def test_one_output_used(device, use, post):
    c = _inputs(device, 21, 520, torch.bfloat16, post=post, gate="channel" if post else "none")
    _compare(c, "layer", 1.0, use)


@pytest.mark.parametrize("device", DEVICES)
def test_many_rows(device):
    """More rows than the workgroups of the backward hold at once, and a large common offset."""
    for rows, width, kind in ((9001, 72, "layer"), (5000, 1032, "rms")):
        _compare(_inputs(device, rows, width, torch.float32, seed=4), kind, 1.0)
    x = torch.randn(64, 1000, generator=torch.Generator().manual_seed(0)).to(device) + 1000.0
    w = torch.ones(1000, device=device)
    y, _ = ops.block_norm(x, kind="layer", pre_weight=w, eps=EPS)
    ref = torch.nn.functional.layer_norm(x.double(), (1000,), eps=EPS)
    # x - mean loses 2^-24 of the mean (1000) twice: 1.2e-4 against a standard deviation of one
    assert (y.double() - ref).abs().max() <= 4 * 1000 * U32 + 64 * U32


@pytest.mark.parametrize("device", DEVICES)
def test_rows_without_spread_and_specials(device):
    """Constant rows (variance zero), rows of zeros, and rows that hold NaN or infinity, which stay theirs."""
    x = torch.zeros(4, 640, device=device)
    x[1] = 3.0
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    w, b = torch.ones(640, device=device), torch.full((640,), 0.5, device=device)
    y, s = ops.block_norm(x, torch.zeros_like(x), kind="layer", pre_weight=w, pre_bias=b, eps=EPS)
    assert torch.equal(y[:2], torch.full_like(y[:2], 0.5)) and y[2].isnan().all() and y[3].isnan().any()
    assert torch.equal(s[:2], x[:2]) and s[2].isnan().sum() == 1


@pytest.mark.parametrize("device", DEVICES)
def test_layouts_and_shapes(device):
    """Strided and shifted inputs, more dimensions, a batch of no rows."""
    c = _inputs(device, 24, 264, torch.bfloat16)
    want = _run(c, "rms", 1.0)
    wide = torch.zeros(24, 300, dtype=torch.bfloat16, device=device)
    wide[:, 3:267] = c["h"]
    odd = torch.zeros(24 * 264 + 1, dtype=torch.bfloat16, device=device)[1:].view(24, 264).copy_(c["residual"])
    y, s = ops.block_norm(wide[:, 3:267].view(24, 264), odd, kind="rms", eps=EPS, **{k: c[k] for k in NAMES[2:]})
    assert torch.allclose(y.float(), want[0].float(), rtol=2 ** -7, atol=1e-6) and y.shape == (24, 264)
    y3, s3 = ops.block_norm(c["h"].view(2, 3, 4, 264), c["residual"].view(2, 3, 4, 264), kind="rms", eps=EPS,
                            **{k: c[k] for k in NAMES[2:]})
    assert torch.equal(y3.view(24, 264), want[0]) and torch.equal(s3.view(24, 264), want[1])
    e = _inputs(device, 1, 264, torch.float32)
    h = torch.zeros(0, 264, device=device, requires_grad=True)
    w = e["pre_weight"].requires_grad_(True)
    y, s = ops.block_norm(h, h, pre_weight=w)
    (y.sum() + s.sum()).backward()
    assert y.shape == (0, 264) and h.grad.shape == (0, 264) and not w.grad.any()
    y, s = ops.block_norm(c["h"])
    assert y is None and torch.equal(s, c["h"])


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x = torch.randn(4, 16, device=device)
    w = torch.ones(16, device=device)
    bad = [
        (dict(kind="batch", pre_weight=w), ValueError),
        (dict(pre_weight=w[:8]), ValueError),
        (dict(pre_bias=w), ValueError),
        (dict(post_bias=w, pre_weight=w), ValueError),
        (dict(pre_weight=w.view(4, 4)), ValueError),
        (dict(gate=w[:2], pre_weight=w), ValueError),
        (dict(gate=torch.ones(4, 16, device=device)), ValueError),
        (dict(residual=torch.zeros(4, 8, device=device), pre_weight=w), ValueError),
        (dict(residual=x.bfloat16(), pre_weight=w), TypeError),
        (dict(pre_weight=w.bfloat16()), TypeError),
        (dict(pre_weight=w, post_weight=w.double()), TypeError),
    ]
    for kw, err in bad:
        with pytest.raises(err):
            ops.block_norm(x, **kw)
    with pytest.raises(TypeError):
        ops.block_norm(torch.ones(4, 16, dtype=torch.int32, device=device), pre_weight=w)
    if device == "cuda":
        with pytest.raises(ValueError):
            ops.block_norm(torch.ones(2, 8200, device=device), pre_weight=torch.ones(8200, device=device))
        with pytest.raises(ValueError):
            ops.block_norm(x, pre_weight=w.cpu())
        with pytest.raises(TypeError):
            ops.block_norm(x.double(), pre_weight=w.double())


def test_gradients_against_differences():
    c = _inputs("cpu", 5, 12, torch.float64, gate="channel")
    ts = [c[k].requires_grad_(True) for k in NAMES]

    def f(*a):
        d = dict(zip(NAMES, a))
        return ops.block_norm(d.pop("h"), d.pop("residual"), kind="layer", scale=0.3, eps=EPS, **d)

    torch.autograd.gradcheck(f, ts)


@pytest.mark.gpu
def test_gradients_against_differences_gpu():
    """fp32 central differences of a weighted sum along random directions, one for each input."""
    c = _inputs("cuda", 6, 40, torch.float32, gate="channel")
    _, _, g = _run(c, "layer", 0.3)
    for k in NAMES:
        d = torch.randn_like(c[k])

        def loss(t):
            cc = {n: (t if n == k else c[n]) for n in NAMES}
            y, s = ops.block_norm(cc["h"], cc["residual"], kind="layer", scale=0.3, eps=EPS, **{n: cc[n] for n in NAMES[2:]})
            return ((y.double() * c["dy"]).sum() + (s.double() * c["ds"]).sum()).item()

        e = 2.0 ** -7
        num = (loss(c[k] + e * d) - loss(c[k] - e * d)) / (2 * e)
        ana = (g[k].double() * d).sum().item()
        # a loss of up to 240 terms of size 10, each with some 32 roundings, over 2 e: 0.02 at most; the
        # third derivative's part is e^2 of a value of the gradient's own size
        assert abs(num - ana) <= 0.02 + 0.02 * abs(ana), k


@pytest.mark.gpu
def test_repeatable_streams_and_graphs():
    c = _inputs("cuda", 3000, 1280, torch.bfloat16, gate="scalar")
    a, b = _run(c, "layer", 0.5), _run(c, "layer", 0.5)
    assert torch.equal(a[0], b[0]) and all(torch.equal(a[2][k], b[2][k]) for k in a[2])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        d = _run(c, "layer", 0.5)
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a[2][k], d[2][k]) for k in a[2])
    # forward and backward in one graph, replayed on new data between eager calls
    leaf = {k: c[k].clone().requires_grad_(True) for k in NAMES}

    def step():
        y, s = ops.block_norm(leaf["h"], leaf["residual"], kind="layer", scale=0.5, eps=EPS, **{k: leaf[k] for k in NAMES[2:]})
        return [y, s, *torch.autograd.grad((y, s), list(leaf.values()), (c["dy"], c["ds"]))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(3):
        new = _inputs("cuda", 3000, 1280, torch.bfloat16, gate="scalar", seed=10 + k)
        with torch.no_grad():
            for n in NAMES:
                leaf[n].copy_(new[n])
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(outs, step()):
            assert torch.equal(x, y)
        torch.cuda.synchronize()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("need", [("h",), ("residual",), ("gate",), ("pre_weight",), ("post_bias", "pre_bias"), ("h", "post_weight")])
def test_some_gradients_only(device, need):
    c = _inputs(device, 40, 520, torch.bfloat16)
    _, _, want = _run(c, "layer", 0.7)
    t = {k: c[k].clone().requires_grad_(k in need) for k in NAMES}
    y, s = ops.block_norm(t["h"], t["residual"], kind="layer", scale=0.7, eps=EPS, **{k: t[k] for k in NAMES[2:]})
    outs = [(o, g) for o, g in ((y, c["dy"]), (s, c["ds"])) if o.requires_grad]
    assert len(outs) == (1 if need == ("pre_weight",) else 2)  # s does not depend on the norm before the next block
    for k, g in zip(need, torch.autograd.grad([o for o, _ in outs], [t[k] for k in need], [g for _, g in outs])):
        assert torch.equal(g, want[k])
    if device == "cuda":
        y, s = ops.block_norm(t["h"], t["residual"], kind="layer", scale=0.7, eps=EPS, **{k: t[k] for k in NAMES[2:]})
        with pytest.raises(RuntimeError, match="again"):
            torch.autograd.grad(y, [t[need[0]]], c["dy"], create_graph=True)


@pytest.mark.parametrize("device", DEVICES)
def test_broadcast_residual_and_stream_used_twice(device):
    c = _inputs(device, 12, 264, torch.float32)
    r = c["residual"][:1].clone().requires_grad_(True)
    h = c["h"].clone().requires_grad_(True)
    y, s = ops.block_norm(h, r.expand(12, 264), kind="rms", pre_weight=c["pre_weight"], eps=EPS)
    y2, s2 = ops.block_norm(y, s, kind="rms", pre_weight=c["pre_weight"], eps=EPS)
    gh, gr = torch.autograd.grad((y2, s2), (h, r), (c["dy"], c["ds"]))
    hd, rd = h.detach().double().requires_grad_(True), r.detach().double().requires_grad_(True)
    w = c["pre_weight"].double()
    a, b = block_norm_ref(hd, rd.expand(12, 264), False, None, None, None, 1.0, w, None, EPS)
    a, b = block_norm_ref(a, b, False, None, None, None, 1.0, w, None, EPS)
    dh, dr = torch.autograd.grad((a, b), (hd, rd), (c["dy"].double(), c["ds"].double()))
    # a few hundred fp32 roundings of values of the gradients' size
    assert ((gh.double() - dh).norm() / dh.norm()).item() <= 1e-5 and ((gr.double() - dr).norm() / dr.norm()).item() <= 1e-5


@pytest.mark.gpu
def test_rows_past_32_bits():
    rows, width = 270000, 8192
    if torch.cuda.mem_get_info()[0] < 40e9:
        pytest.skip("needs 40 GB")
    h = torch.zeros(rows, width, device="cuda", dtype=torch.bfloat16)
    ends = torch.tensor([0, 1, rows // 2, rows - 2, rows - 1], device="cuda")
    c = _inputs("cuda", 5, width, torch.bfloat16)
    h[ends] = c["h"]
    h.requires_grad_(True)
    w = c["pre_weight"].requires_grad_(True)
    y, _ = ops.block_norm(h, kind="rms", pre_weight=w, eps=EPS)
    dy = torch.zeros_like(y)
    dy[ends] = c["dy"]
    dh, dw = torch.autograd.grad(y, (h, w), dy)
    hs = c["h"].clone().requires_grad_(True)
    ys, _ = ops.block_norm(hs, kind="rms", pre_weight=w, eps=EPS)
    dhs, dws = torch.autograd.grad(ys, (hs, w), c["dy"])
    assert torch.equal(y[ends], ys) and torch.equal(dh[ends], dhs) and not dh[2:rows // 2].any()
    assert ((dw.double() - dws.double()).norm() / dws.double().norm()).item() <= 2.0 ** -8  # another order, rounded


@pytest.mark.gpu
def test_main_grad_takes_the_sums():
    c = _inputs("cuda", 300, 520, torch.bfloat16)
    ts = {k: c[k].clone().requires_grad_(True) for k in NAMES}
    for k in NAMES[2:]:
        ts[k].main_grad = torch.full(ts[k].shape, 2.0, device="cuda")
    y, s = ops.block_norm(ts["h"], ts["residual"], kind="layer", eps=EPS, **{k: ts[k] for k in NAMES[2:]})
    torch.autograd.backward((y, s), (c["dy"], c["ds"]))
    _, _, rg = _ref(c, "layer", 1.0)
    for k in NAMES[2:]:
        assert ts[k].grad is None
        err = (ts[k].main_grad.double().cpu() - 2.0 - rg[k]).norm() / rg[k].norm()
        assert err <= 1e-5, k  # fp32 sums: no 16-bit rounding enters


@pytest.mark.gpu
@pytest.mark.parametrize("main_grad", [False, True])
def test_capture_beside_a_live_graph_is_refused(main_grad):
    """Refused before anything of it is recorded; without the earlier graph the same capture works."""
    h = torch.nn.Parameter(torch.randn(8, 64, device="cuda"))
    w = torch.nn.Parameter(torch.ones(64, device="cuda"))
    if main_grad:
        w.main_grad = torch.zeros(64, device="cuda")
    live = ops.block_norm(h, pre_weight=w)
    for _ in range(2):
        torch.cuda.synchronize()
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            keep = torch.zeros(4, device="cuda")
            with torch.no_grad():
                y = ops.block_norm(h, pre_weight=w)
            if live is not None:
                with pytest.raises(RuntimeError, match="earlier autograd graph"):
                    ops.block_norm(h, pre_weight=w)
            else:
                torch.autograd.grad(ops.block_norm(h, pre_weight=w)[0], [h], torch.ones_like(h))
        live = None
    del keep, y


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", NAMES)
@pytest.mark.parametrize("leaf", [False, True])
@pytest.mark.parametrize("main_grad", [False, True])
def test_forward_mode_is_right_or_refused(device, which, leaf, main_grad):
    """A tangent is never dropped: the CPU's operations carry it, the kernels refuse the call."""
    import torch.autograd.forward_ad as fwd

    c = _inputs(device, 5, 16, torch.float32)
    t = {k: c[k].clone().requires_grad_(leaf) for k in NAMES}
    with fwd.dual_level():
        t[which] = fwd.make_dual(t[which], torch.ones_like(t[which]))
        if main_grad:
            t["pre_weight"].main_grad = torch.zeros(16, device=device)

        def call():
            y, s = ops.block_norm(t["h"], t["residual"], kind="layer", eps=EPS, **{k: t[k] for k in NAMES[2:]})
            return fwd.unpack_dual(y).tangent

        if device == "cpu":  # zero where a layer norm takes a constant away
            got = call()
            assert got is not None and (got.any() or which in ("h", "residual"))
        else:
            with pytest.raises(NotImplementedError):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call()
    if device == "cuda":
        rest = {k: c[k] for k in NAMES if k != which}
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.func.jvp(lambda v: ops.block_norm(**rest, **{which: v}, eps=EPS), (c[which],), (torch.ones_like(c[which]),))


@pytest.mark.gpu
@pytest.mark.parametrize("main_grad", [False, True])
def test_capture_of_a_strided_leaf_beside_a_live_graph_is_refused(main_grad):
    """The leaf itself is looked at, not the contiguous copy that the kernel reads."""
    h = torch.nn.Parameter(torch.randn(64, 8, device="cuda").t())
    w = torch.ones(64, device="cuda")
    if main_grad:
        w.main_grad = torch.zeros(64, device="cuda")
    assert not h.is_contiguous()
    live = h * 1
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        keep = torch.zeros(4, device="cuda")
        with pytest.raises(RuntimeError, match="earlier autograd graph"):
            ops.block_norm(h, pre_weight=w)
    del live, keep


@pytest.mark.gpu
def test_strided_and_expanded_weights_beside_main_grad():
    """A gate that is one value expanded, a bias that is a column of something wider."""
    c = _inputs("cuda", 40, 264, torch.bfloat16)

    def run(main_grad):
        g = c["gate"][:1].clone().requires_grad_(True)
        wide = torch.stack([c["pre_bias"], c["post_bias"]], 1).requires_grad_(True)
        w = c["pre_weight"].clone().requires_grad_(True)
        if main_grad:
            w.main_grad = torch.zeros(264, device="cuda")
        y, s = ops.block_norm(c["h"], c["residual"], kind="layer", post_weight=c["post_weight"], post_bias=wide[:, 1],
                              gate=g.expand(264), pre_weight=w, pre_bias=wide[:, 0], eps=EPS)
        torch.autograd.backward((y, s), (c["dy"], c["ds"]))
        return y, s, g.grad, wide.grad, (w.main_grad if main_grad else w.grad)

    for a, b in zip(run(True)[:4], run(False)):
        assert torch.equal(a, b)
    w32, w16 = run(True)[4], run(False)[4]
    assert torch.equal(w32.bfloat16(), w16)  # the same sums, rounded once


@pytest.mark.gpu
@pytest.mark.parametrize("width", [1000, 1001])
def test_a_scalar_gate_sums_its_columns_in_64_bits(width):
    """dgate = sum of ds h over 3001 rows: every other column adds up to 3001 (1 + 2^-20), the ones between to -3001,
    which needs 32 bits.  A lane's own sum of three rows is exact in fp32; so is all behind it in 64 bits."""
    h = torch.ones(3001, width, device="cuda")
    gate = torch.ones(1, device="cuda", requires_grad=True)
    ds = torch.full_like(h, -1.0)
    ds[:, ::2] = 1 + 2.0 ** -20
    _, s = ops.block_norm(h, torch.zeros_like(h), gate=gate)
    (dg,) = torch.autograd.grad(s, gate, ds)
    want = ds.double().sum().item()
    assert abs(dg.item() - want) <= U32 * abs(want) * 1.01


@pytest.mark.gpu
def test_weight_gradients_round_once_behind_the_rows():
    """fp32 column sums of 3001 rows: a chain of three fp32 additions a lane, the rest in 64 bits and one rounding."""
    c = _inputs("cuda", 3001, 1001, torch.float32, gate="scalar", seed=2)
    _, _, g = _run(c, "layer", 0.5)
    _, _, rg = _ref(c, "layer", 0.5)
    for k in NAMES[2:]:
        # random signs: a term of the sums is off by some 8 roundings, a lane's chain by 3, together some 4 U of the
        # sums' own 2-norm; 6 times that.  The gate's single sum is as large as the 2-norm of the columns' sums.
        size = rg[k].norm().item() if k != "gate" else rg["post_weight"].norm().item() / abs(c["gate"].item())
        assert (g[k].double().cpu() - rg[k]).norm().item() <= 6 * 4 * U32 * size, k
