"""Linear with bias, activation and residual in the epilogue (ops/linear_act.py, csrc/linear_act_*.hip)
against 64 bits.

Tolerances, element by element.  A sum of k products in fp32 in any order is off by at most k 2^-24
times the sum of the products' magnitudes.  The activations have slopes of at most 1.13 and are
themselves computed to 2e-6 of |z| + 1e-7; an output is rounded once, by u = eps / 2 of its type.  In
the backward z and dz are kept in x's type: dz is off by u |dz| + |dy| (C u |z| + 4e-6), C bounding
the activation's second derivative (0.8 gelu and its tanh form 0.9, silu 0.5, relu 0), and dx, dW and
db by the sums of those errors over the products' other factors.
"""
import pytest
import torch

from scaletorch_amd import ops
from scaletorch_amd.models.gpt import GPT, GPTConfig
from scaletorch_amd.ops.linear_act import linear_act_ref

U32 = 2.0 ** -24
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
CURVE = {"none": 0.0, "relu": 0.0, "gelu": 0.8, "gelu_tanh": 0.9, "silu": 0.5}


def _inputs(device, m, k, n, dtype, bias=True, residual=True, rdtype=None, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)

    def make(*shape, std=1.0, dt=dtype):
        return (torch.randn(*shape, generator=g) * std).to(dt).to(device)

    return dict(x=make(m, k, std=scale), w=make(n, k, std=k ** -0.5), b=make(n, std=0.5) if bias else None,
                r=make(m, n, std=2.0, dt=rdtype or dtype) if residual else None, dy=make(m, n, dt=rdtype if residual and rdtype else dtype))


def _run(c, act, f=ops.linear_act):
    t = {k: None if c[k] is None else c[k].detach().clone().requires_grad_(True) for k in "xwbr"}
    y = f(t["x"], t["w"], t["b"], t["r"], act)
    some = [k for k in "xwbr" if t[k] is not None]
    return y, dict(zip(some, torch.autograd.grad(y, [t[k] for k in some], c["dy"])))


def _within(got, ref, bound, u, what):
    got, ref, bound = got.detach().double().cpu(), ref.detach().double(), bound.detach()
    tiny = 2.0 ** -24 if u == 2.0 ** -11 else 2.0 ** -60
    over = (got - ref).abs() - (bound + u * (ref.abs() + bound) * 1.01 + tiny)
    assert (over <= 0).all(), f"{what}: {over.max().item():.3g} past the bound"


def _compare(c, act):
    y, g = _run(c, act)
    d = {k: None if v is None else v.double().cpu() for k, v in c.items()}
    ry, rg = _run(d, act, lambda x, w, b, r, a: linear_act_ref(x, w, b, r, a))
    u = torch.finfo(c["x"].dtype).eps / 2 if c["x"].dtype != torch.float32 else U32
    x, w, dy = d["x"], d["w"], d["dy"]
    (m, k), n = x.shape, w.shape[0]
    z = x @ w.t() + (0 if d["b"] is None else d["b"])
    ez = (k + 4) * U32 * (x.abs() @ w.abs().t() + (0 if d["b"] is None else d["b"].abs()))
    ey = 1.13 * ez + 2e-6 * z.abs() + 1e-7 + 2 * U32 * (0 if d["r"] is None else d["r"].abs())
    _within(y, ry, ey, torch.finfo(y.dtype).eps / 2, "y")
    zz = z.clone().requires_grad_(True)
    from scaletorch_amd.ops.linear_act import _act_ref
    slope = torch.autograd.grad(_act_ref(zz, act).sum(), zz)[0]
    dz = dy * slope
    edz = u * dz.abs() + dy.abs() * (CURVE[act] * (u * z.abs() + ez) + 4e-6)
    if act == "none":
        edz = (u if c["dy"].dtype != c["x"].dtype else 0.0) * dz.abs()
    if act == "relu":  # within z's error of zero the slope may be the other one
        edz = edz + dy.abs() * (z.abs() <= ez).double()
    if c["x"].dtype == torch.float16:
        edz = edz + 2.0 ** -24
    _within(g["x"], rg["x"], edz @ w.abs() + (n + 4) * U32 * ((dz.abs() + edz) @ w.abs()), u, "dx")
    _within(g["w"], rg["w"], edz.t() @ x.abs() + (m + 4) * U32 * ((dz.abs() + edz).t() @ x.abs()), u, "dw")
    if "b" in g:
        _within(g["b"], rg["b"], edz.sum(0) + (m + 4) * U32 * dz.abs().sum(0), u, "db")
    if "r" in g:
        assert torch.equal(g["r"], c["dy"])
    return y, g


SHAPES = [(1, 8, 4), (1, 1, 1), (3, 33, 7), (16, 256, 128), (17, 1000, 264), (33, 72, 40), (64, 520, 1000), (65, 64, 64),
          (65, 65, 65), (130, 1000, 200), (300, 136, 8), (257, 100, 333), (129, 24, 2048), (1000, 520, 264)]
# few rows: 16 and 32 columns a workgroup, ends of k and of the columns inside one
SHAPES += [(2, 40, 24), (4, 72, 8200), (5, 1000, 264), (9, 2056, 1000), (16, 1032, 8200)]
# a few more rows, inner sizes of whole steps
WIDE = [(512, 256, 512), (1025, 320, 776), (777, 1024, 264)]
LARGE = [(4096, 512, 4104), (2056, 2048, 2568), (8200, 64, 8192), (16448, 1280, 1288), (300, 8192, 1024)]
# the 256 x 256 tiles: one, two and three steps of k, cut tiles in y, dx and dW, whole ones of ragged edges
LARGE += [(5128, 64, 8712), (3336, 128, 8456), (1288, 192, 8968), (4200, 1984, 4104), (6001, 1320, 5120), (4100, 1024, 4096), (5000, 1288, 5056)]
# the smaller tiles, each in turn: 128 x 128 in y, 64 x 128 in dx, in dW, in dW with k split, 128 x 128 in dx, in dW
TILES = [(4104, 136, 3080), (2056, 776, 520), (520, 776, 2312), (4104, 776, 1352), (2056, 1544, 328), (328, 1544, 2056)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", SHAPES + WIDE)
def test_shapes(device, dtype, m, k, n):
    _compare(_inputs(device, m, k, n, dtype), "gelu")


@pytest.mark.gpu
@pytest.mark.parametrize("act,residual,rdtype,dtype", [("gelu", True, torch.float32, torch.bfloat16), ("none", True, None, torch.float16),
                                                       ("silu", True, None, torch.bfloat16), ("gelu_tanh", False, None, torch.bfloat16)])
@pytest.mark.parametrize("m,k,n", LARGE + TILES)
def test_large(m, k, n, act, residual, rdtype, dtype):
    """Against fp32 products on the GPU (the library's, checked at 64 bits where that is quick), whole tensors."""
    c = _inputs("cuda", m, k, n, dtype, True, residual, rdtype, seed=m)
    y, g = _run(c, act)
    d = {k: None if v is None else v.double() for k, v in c.items()}
    ry, rg = _run(d, act, lambda x, w, b, r, a: linear_act_ref(x, w, b, r, a))
    u = torch.finfo(dtype).eps / 2
    for got, ref, uu in ((y, ry, torch.finfo(y.dtype).eps / 2), (g["x"], rg["x"], 3 * u), (g["w"], rg["w"], 3 * u), (g["b"], rg["b"], 3 * u)):
        ref = ref.detach()
        # the 2-norm: one rounding of y; z's, dz's and the result's own in the gradients; fp32 sums of up to
        # 16448 terms of random signs, some sqrt(16448) 2^-24 of the result
        err = ((got.detach().double() - ref).norm() / ref.norm()).item()
        assert err <= uu + 2e-5, (got.shape, err)
        # and no element further off than six times that of the largest
        assert (got.detach().double() - ref).abs().max() <= 6 * (uu + 2e-5) * ref.abs().max()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("residual", [None, "same", "fp32"])
def test_each_part(device, act, bias, residual):
    for k, (dtype, (m, kk, n)) in enumerate(((torch.bfloat16, (70, 96, 136)), (torch.float16, (9, 40, 24)),
                                             (torch.bfloat16, (131, 77, 35)), (torch.float16, (515, 128, 264)))):
        c = _inputs(device, m, kk, n, dtype, bias, residual is not None, torch.float32 if residual == "fp32" else None,
                    seed=k, scale=2.0)
        _compare(c, act)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
def test_activation_range(device, act):
    """z from -60 to 60 by an identity weight, and zero, infinities and NaN."""
    z = torch.cat([torch.linspace(-60, 60, 4096), torch.linspace(-6, 6, 4096), torch.tensor([0.0, -0.0])])
    z = torch.nn.functional.pad(z, (0, 8200 - z.numel())).to(torch.bfloat16).view(-1, 8).to(device)
    w = torch.eye(8, dtype=torch.bfloat16, device=device)
    t = z.clone().requires_grad_(True)
    y = ops.linear_act(t, w, residual=torch.zeros_like(z, dtype=torch.float32), activation=act)
    (dx,) = torch.autograd.grad(y, t, torch.ones_like(y))
    r = z.double().cpu().requires_grad_(True)
    from scaletorch_amd.ops.linear_act import _act_ref
    ry = _act_ref(r, act)
    (rdx,) = torch.autograd.grad(ry, r, torch.ones_like(ry))
    assert ((y.double().cpu() - ry).abs() <= 2e-6 * r.abs() + 1e-7).all()
    assert ((dx.double().cpu() - rdx).abs() <= 2.0 ** -8 * rdx.abs() * 1.01 * 2 + 4e-6).all()
    special = torch.tensor([[float("inf"), float("nan"), -float("inf"), 1e30, -1e30, 2.0, 3.0, 4.0]] * 3, device=device)
    one = torch.ones(1, 1, device=device).bfloat16()
    got = ops.linear_act(special.bfloat16().view(-1, 1), one, activation=act).float().view(3, 8)
    assert got[0, 0] == float("inf") and got[0, 1].isnan() and got[0, 3] > 9e29 and got[0, 4] == 0 and (got[0, 5:] > 1.5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows", [2, 300])
def test_sums_past_fp16_range(act, rows):
    """z = 262144 and -262144: finite in y (fp32), beyond what fp16 keeps for the backward.  Every value
    here is exact: slopes of 1 and 0, and sums of powers of two."""
    x = torch.full((rows, 1024), 256.0, device="cuda").half().requires_grad_(True)
    w = torch.ones(8, 1024, device="cuda").half()
    w[1::2] = -1
    w.requires_grad_(True)
    y = ops.linear_act(x, w, residual=torch.zeros(rows, 8, device="cuda"), activation=act)
    assert (y[:, ::2] == 262144.0).all() and (y[:, 1::2] == 0).all()
    dx, dw = torch.autograd.grad(y, [x, w], torch.full_like(y, 2.0 ** -10))
    assert (dx == 2.0 ** -8).all()
    assert (dw[::2] == rows / 4).all() and (dw[1::2] == 0).all()


@pytest.mark.gpu
def test_dimensions_past_the_limit_are_refused():
    x = torch.empty(2 ** 31 - 1, 1, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="at most"):
        ops.linear_act(x, torch.ones(1, 1, device="cuda", dtype=torch.bfloat16))


@pytest.mark.parametrize("device", DEVICES)
def test_layouts(device):
    """More dimensions, padded rows, shifted starts, columns of a wider tensor, a transposed weight, no rows."""
    c = _inputs(device, 24, 72, 40, torch.bfloat16)
    want, grads = _run(c, "silu")
    y = ops.linear_act(c["x"].view(2, 3, 4, 72), c["w"], c["b"], c["r"].view(2, 3, 4, 40), "silu")
    assert y.shape == (2, 3, 4, 40) and torch.equal(y.view(24, 40), want)
    wide = torch.randn(24, 100, device=device).bfloat16()
    wide[:, 5:77] = c["x"]
    odd = torch.zeros(40 * 72 + 1, dtype=torch.bfloat16, device=device)[1:].view(40, 72).copy_(c["w"])
    for x, w in ((wide[:, 5:77], c["w"]), (c["x"], odd), (c["x"], c["w"].t().contiguous().t()),
                 (c["x"].t().contiguous().t(), c["w"])):
        d = dict(c, x=x, w=w)
        x, w = (v.detach().requires_grad_(True) for v in (x, w))
        y = ops.linear_act(x, w, c["b"], c["r"], "silu")
        # another order of the same fp32 sums, rounded once
        assert (y.float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()
        dx, dw = torch.autograd.grad(y, (x, w), c["dy"])
        for a, b in ((dx, grads["x"]), (dw, grads["w"])):
            assert (a.float() - b.float()).abs().max() <= 2.0 ** -6 * b.float().abs().max()
    y = ops.linear_act(c["x"][:0], c["w"], c["b"], activation="gelu")
    assert y.shape == (0, 40)
    e = _inputs(device, 1, 72, 40, torch.bfloat16)
    y = ops.linear_act(e["x"][0], e["w"], e["b"], e["r"][0], "relu")
    assert y.shape == (40,)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x, w, b = (torch.zeros(s, dtype=torch.bfloat16, device=device) for s in ((4, 16), (8, 16), (8,)))
    bad = [
        ((x, w, b, None, "swish"), ValueError),
        ((x, w.t(), None, None, "none"), ValueError),
        ((x, w, b[:4], None, "none"), ValueError),
        ((x, w, b, x, "none"), ValueError),
        ((x, w.view(2, 4, 16), b, None, "none"), ValueError),
        ((x, w.float(), None, None, "none"), TypeError),
        ((x, w, b.half(), None, "none"), TypeError),
        ((x, w, b, torch.zeros(4, 8, device=device, dtype=torch.float16), "none"), TypeError),
        ((x.int(), w.int(), None, None, "none"), TypeError),
    ]
    for args, err in bad:
        with pytest.raises(err):
            ops.linear_act(*args)
    if device == "cuda":
        with pytest.raises(TypeError):
            ops.linear_act(x.float(), w.float())
        with pytest.raises((ValueError, RuntimeError)):
            ops.linear_act(x, w.cpu())


def test_gradients_against_differences():
    g = torch.Generator().manual_seed(0)
    x, w, b, r = (torch.randn(s, generator=g, dtype=torch.float64).requires_grad_(True) for s in ((3, 5), (4, 5), (4,), (3, 4)))
    for act in ("gelu", "gelu_tanh", "silu"):
        torch.autograd.gradcheck(lambda *a: ops.linear_act(*a, activation=act), (x, w, b, r))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_gradients_against_differences_gpu(act):
    """Central differences of the fp32 output along one direction of the bias."""
    c = _inputs("cuda", 70, 96, 136, torch.bfloat16, rdtype=torch.float32)
    _, g = _run(c, act)
    e = 0.125  # an exact bf16 change of a bias that is kept in eighths
    c["b"] = (c["b"].float() * 8).round().div(8).bfloat16()
    _, g = _run(c, act)
    f = lambda b: (ops.linear_act(c["x"], c["w"], b, c["r"], act).double() * c["dy"]).sum().item()  # noqa: E731
    d = torch.sign(c["b"].float())
    num = (f((c["b"].float() + e * d).bfloat16()) - f((c["b"].float() - e * d).bfloat16())) / (2 * e)
    ana = (g["b"].double() * d).sum().item()
    # 9520 terms, each with a third-derivative part of at most e^2 / 6 * 2 |dy| and roundings of z and dz of
    # 2^-8: independent signs, so some 6 sqrt(9520) (0.006 + 0.008)
    assert abs(num - ana) <= 6 * 9520 ** 0.5 * 0.014


@pytest.mark.gpu
def test_repeatable_streams_graphs_and_no_grad():
    for shape in ((1000, 520, 264), (33, 72, 40), (2048, 512, 1280)):
        c = _inputs("cuda", *shape, torch.bfloat16)
        a, b = _run(c, "gelu"), _run(c, "gelu")
        assert torch.equal(a[0], b[0]) and all(torch.equal(a[1][k], b[1][k]) for k in a[1])
        with torch.no_grad():
            assert torch.equal(ops.linear_act(c["x"], c["w"], c["b"], c["r"], "gelu"), a[0])
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            d = _run(c, "gelu")
        torch.cuda.current_stream().wait_stream(st)
        assert all(torch.equal(a[1][k], d[1][k]) for k in a[1])
    leaf = {k: c[k].clone().requires_grad_(True) for k in "xwbr"}

    def step():
        y = ops.linear_act(leaf["x"], leaf["w"], leaf["b"], leaf["r"], "gelu")
        return [y, *torch.autograd.grad(y, list(leaf.values()), c["dy"])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs, each with its own workspaces
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for k in range(3):
        new = _inputs("cuda", 2048, 512, 1280, torch.bfloat16, seed=10 + k)
        with torch.no_grad():
            for n in "xwbr":
                leaf[n].copy_(new[n])
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, outs in graphs:
            for x, y in zip(outs, step()):
                assert torch.equal(x, y)
        torch.cuda.synchronize()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("need", ["x", "w", "b", "r", "xw", "wb", "br"])
def test_some_gradients_only(device, need):
    c = _inputs(device, 70, 96, 136, torch.bfloat16)
    _, want = _run(c, "gelu")
    t = {k: c[k].clone().requires_grad_(k in need) for k in "xwbr"}
    y = ops.linear_act(t["x"], t["w"], t["b"], t["r"], "gelu")
    for k, g in zip(need, torch.autograd.grad(y, [t[k] for k in need], c["dy"])):
        assert torch.equal(g, want[k])
    if device == "cuda":
        y = ops.linear_act(t["x"], t["w"], t["b"], t["r"], "gelu")
        with pytest.raises(RuntimeError, match="again"):
            torch.autograd.grad(y, [t[need[0]]], c["dy"], create_graph=True)


@pytest.mark.parametrize("device", DEVICES)
def test_broadcast_and_expanded_operands(device):
    """A bias and residual expanded over rows, a gradient that is one value expanded."""
    c = _inputs(device, 40, 64, 24, torch.bfloat16)
    r = c["r"][:1].clone().requires_grad_(True)
    y = ops.linear_act(c["x"], c["w"], c["b"], r.expand(40, 24), "silu")
    want = ops.linear_act(c["x"], c["w"], c["b"], r.detach().repeat(40, 1), "silu")
    assert torch.equal(y, want)
    y.float().sum().backward()
    assert torch.equal(r.grad, torch.full_like(r, 40.0))
    x = c["x"][:1].expand(40, 64).detach().requires_grad_(True)
    y = ops.linear_act(x, c["w"])
    assert torch.equal(y[0], y[39])
    y.sum().backward()
    assert torch.equal(x.grad[0], x.grad[39])


@pytest.mark.gpu
def test_outputs_past_32_bits():
    """An output of more than 2^31 elements and its gradients, at both ends."""
    m, k, n = 70000, 64, 32776
    if torch.cuda.mem_get_info()[0] < 30e9:
        pytest.skip("needs 30 GB")
    g = torch.Generator("cuda").manual_seed(0)
    x, w = (torch.randn(s, k, device="cuda", generator=g).bfloat16().requires_grad_(True) for s in (m, n))
    y = ops.linear_act(x, w, activation="relu")
    dy = torch.zeros_like(y)
    ends = [0, 1, m // 2, m - 2, m - 1]
    dy[ends] = 1.0
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    xd, wd = x.detach()[ends].double(), w.detach().double()
    z = xd @ wd.t()
    assert ((y[ends].double() - z.clamp_min(0)).abs() <= 2.0 ** -8 * z.abs() + 1e-4).all()
    dz = (z > 0).double()
    # an element whose z is within fp32's error of zero may count the other way: none is expected
    assert ((dx[ends].double() - dz @ wd).norm() / (dz @ wd).norm()).item() <= 2.0 ** -8
    assert not dx[2:m // 2].any()
    assert ((dw.double() - dz.t() @ xd).norm() / (dz.t() @ xd).norm()).item() <= 2.0 ** -8


@pytest.mark.gpu
def test_main_grad_takes_the_sums():
    c = _inputs("cuda", 512, 256, 512, torch.bfloat16)
    t = {k: c[k].clone().requires_grad_(True) for k in "xwbr"}
    for k in "wb":
        t[k].main_grad = torch.full(t[k].shape, 2.0, device="cuda")
    ops.linear_act(t["x"], t["w"], t["b"], t["r"], "gelu").backward(c["dy"])
    _, g = _run(c, "gelu")
    for k in "wb":
        assert t[k].grad is None
        # the plain gradient is the same sum rounded to bf16
        assert ((t[k].main_grad - 2.0 - g[k].float()).abs() <= 2.0 ** -8 * 1.01 * g[k].float().abs() + 1e-3).all()
    assert torch.equal(t["x"].grad, g["x"]) and torch.equal(t["r"].grad, g["r"])


@pytest.mark.gpu
def test_autocast_casts_as_linear_does():
    x, w, b = (torch.randn(s, device="cuda") for s in ((40, 64), (32, 64), (32,)))
    r = torch.randn(40, 32, device="cuda")
    x.requires_grad_(True)
    w.requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = ops.linear_act(x, w, b, r, "gelu")
    assert y.dtype == torch.float32
    c = dict(x=x.detach().bfloat16(), w=w.detach().bfloat16(), b=b.bfloat16(), r=r, dy=torch.randn(40, 32, device="cuda"))
    want, g = _run(c, "gelu")
    assert torch.equal(y, want)
    dx, dw = torch.autograd.grad(y, (x, w), c["dy"])
    assert dx.dtype == torch.float32 and torch.equal(dx, g["x"].float()) and torch.equal(dw, g["w"].float())


@pytest.mark.gpu
@pytest.mark.parametrize("main_grad", [False, True])
def test_capture_beside_a_live_graph_is_refused(main_grad):
    """Refused before anything of it is recorded; without the earlier graph the same capture works."""
    c = _inputs("cuda", 64, 64, 64, torch.bfloat16)
    x, w = (torch.nn.Parameter(c[k]) for k in "xw")
    if main_grad:
        w.main_grad = torch.zeros(64, 64, device="cuda")
    live = ops.linear_act(x, w, activation="gelu")
    for _ in range(2):
        torch.cuda.synchronize()
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            keep = torch.zeros(4, device="cuda")
            with torch.no_grad():
                y = ops.linear_act(x, w, activation="gelu")
            if live is not None:
                with pytest.raises(RuntimeError, match="earlier autograd graph"):
                    ops.linear_act(x, w, activation="gelu")
            else:
                torch.autograd.grad(ops.linear_act(x, w, activation="gelu"), [x], c["dy"])
        live = None
    del keep, y


# one row of x behind whose last step of k only a part of a step is left (24 of 32, 56 of 64 values), and a last
# tile of one row with the same end, in y and, of the columns, in dx
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m,k,n", [(1, 24, 8), (1, 56, 24), (1, 88, 8200), (1, 4088, 64), (65, 56, 136), (65, 120, 136),
                                   (129, 184, 264), (65, 64, 56), (193, 128, 184), (257, 1016, 2040)])
def test_last_step_of_a_single_row(device, m, k, n):
    _compare(_inputs(device, m, k, n, torch.bfloat16), "gelu")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", "xwbr")
@pytest.mark.parametrize("leaf", [False, True])
@pytest.mark.parametrize("main_grad", [False, True])
def test_forward_mode_is_right_or_refused(device, which, leaf, main_grad):
    """A tangent is never dropped: the CPU's operations carry it, the kernels refuse the call."""
    import torch.autograd.forward_ad as fwd

    c = _inputs(device, 5, 16, 8, torch.bfloat16)
    t = {k: c[k].clone().requires_grad_(leaf) for k in "xwbr"}
    if main_grad:
        t["w"].main_grad = torch.zeros(8, 16, device=device)
    with fwd.dual_level():
        t[which] = fwd.make_dual(t[which], torch.ones_like(t[which]))
        if main_grad and which == "w":
            t["w"].main_grad = torch.zeros(8, 16, device=device)

        def call():
            return fwd.unpack_dual(ops.linear_act(t["x"], t["w"], t["b"], t["r"], "silu")).tangent

        if device == "cpu":
            got = call()
            assert got is not None and got.any()
        else:
            with pytest.raises(NotImplementedError):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call()
    if device == "cuda":
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.func.jvp(lambda v: ops.linear_act(**{**{"x": c["x"], "weight": c["w"]}, {"x": "x", "w": "weight", "b": "bias", "r": "residual"}[which]: v}),
                           (c[which],), (torch.ones_like(c[which]),))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [(1, 8, 4), (65, 65, 65), (777, 1024, 264), (328, 1544, 2056), (4100, 1024, 4096)])
def test_main_grad_sums_in_fp32_and_in_its_own_type(m, k, n, dtype):
    """dW added to an fp32 buffer, which is not rounded to 16 bits, and to a 16-bit one, rounded once; the first
    gradient of a step overwrites."""
    c = _inputs("cuda", m, k, n, dtype, False, False)
    z = c["x"].double() @ c["w"].double().t()
    dz = c["dy"].double() * (z > 0)
    want, size = dz.t() @ c["x"].double(), dz.abs().t() @ c["x"].double().abs()
    far = (z.abs() <= (k + 4) * U32 * (c["x"].double().abs() @ c["w"].double().abs().t())).double()
    # relu keeps dz exact but where z is within its error of zero; then fp32 sums of m terms and the addition of 2
    bound = (m + 4) * U32 * (size + 2) + (far * c["dy"].double().abs()).t() @ c["x"].double().abs()
    for mt in (torch.float32, dtype):
        w = c["w"].clone().requires_grad_(True)
        w.main_grad = torch.full((n, k), 2.0, device="cuda", dtype=mt)
        calls = []
        w._st_grad_ready = calls.append
        u = torch.finfo(mt).eps / 2
        for fresh in (False, True):
            w._st_fresh = fresh
            old = 0.0 if fresh else 2.0
            ops.linear_act(c["x"], w, activation="relu").backward(c["dy"])
            assert ((w.main_grad.double() - old - want).abs() <= bound + 1.01 * u * (want + old).abs()).all()
            assert not w._st_fresh
        assert w.grad is None and calls == [w, w]


@pytest.mark.gpu
def test_main_grad_backward_needs_no_library(monkeypatch):
    """Neither the library's products nor their tuner may run: both break a capture that meets them first."""
    from scaletorch_amd.ops import grad

    def refuse(*a, **k):
        raise AssertionError("the weight gradient went to the tuned products")

    monkeypatch.setattr(grad, "wgrad_into", refuse)
    c = _inputs("cuda", 64, 64, 64, torch.bfloat16)
    w = c["w"].clone().requires_grad_(True)
    w.main_grad = torch.zeros(64, 64, device="cuda")
    ops.linear_act(c["x"], w, c["b"], c["r"], "gelu").backward(c["dy"])
    assert w.main_grad.any()


@pytest.mark.gpu
def test_main_grad_backward_is_captured():
    """Forward and backward with main_grad in a graph without a pass before it, replayed between eager passes."""
    c = _inputs("cuda", 200, 136, 264, torch.bfloat16)
    t = {k: torch.nn.Parameter(c[k]) for k in "xwb"}
    for k in "wb":
        t[k].main_grad = torch.zeros(t[k].shape, device="cuda")

    def step():
        for k in "wb":
            t[k].main_grad.zero_()
        y = ops.linear_act(t["x"], t["w"], t["b"], activation="gelu")
        (dx,) = torch.autograd.grad(y, [t["x"]], c["dy"])
        return y.detach(), dx

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        new = _inputs("cuda", 200, 136, 264, torch.bfloat16, seed=seed + 5)
        with torch.no_grad():
            for k in "xwb":
                t[k].copy_(new[k])
        c["dy"].copy_(new["dy"])
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in (*outs, t["w"].main_grad, t["b"].main_grad)]
        want = [*step(), t["w"].main_grad, t["b"].main_grad]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("main_grad", [False, True])
@pytest.mark.parametrize("held", ["linear", "cast"])
def test_capture_beside_a_live_graph_is_refused_under_autocast(main_grad, held):
    """The leaves are fp32 parameters whose 16-bit copies the operator takes.  Only the refusal is called: nothing of
    it may be recorded."""
    x, w, b = (torch.nn.Parameter(torch.randn(s, device="cuda")) for s in ((64, 64), (32, 64), (32,)))
    if main_grad:
        b.main_grad = torch.zeros(32, device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        live = ops.linear_act(x, w, b, activation="gelu") if held == "linear" else [v.bfloat16() for v in (x, w, b)]
        torch.cuda.synchronize()
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            keep = torch.zeros(4, device="cuda")
            with torch.no_grad():
                y = ops.linear_act(x, w, b, activation="gelu")
            with pytest.raises(RuntimeError, match="earlier autograd graph"):
                ops.linear_act(x, w, b, activation="gelu")
    del live, keep, y


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [3, 500])
def test_tails_are_relative(device, act, dtype, rows):
    """y and dx for z in [-9, 0], relative to the value itself, by an identity weight and an fp32 residual of zeros.

    y = z s: s is a fit or sum of relative error 1e-6 at most times an exponential whose argument a (natural, up to
    z^2 / 2 = 41, and 2 sqrt(2 / pi) (|z| + 0.045 |z|^3) = 67 in the tanh form) is off by 3 roundings of it, its
    constants' included; in the tanh form, whose argument is a longer product, by up to 10."""
    z = -(torch.arange(rows * 8) % 2305).float().div(256).to(dtype).view(rows, 8).to(device)
    w = torch.eye(8, dtype=dtype, device=device)
    x = z.clone().requires_grad_(True)
    y = ops.linear_act(x, w, residual=torch.zeros(rows, 8, device=device), activation=act)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    r = z.double().requires_grad_(True)
    from scaletorch_amd.ops.linear_act import _act_ref
    ry = _act_ref(r, act)
    (rdx,) = torch.autograd.grad(ry, r, torch.ones_like(ry))
    a = {"gelu": r * r / 2, "gelu_tanh": 1.6 * (r.abs() + 0.045 * r.abs() ** 3), "silu": r.abs()}[act].detach()
    rel = 1e-6 + ((10 if act == "gelu_tanh" else 3) * a + 16) * U32
    assert ((y.double() - ry).abs() <= rel * ry.abs() + 1e-30).all()
    # the slope is a sum of two such terms, s and z s'(z), of opposite signs; rounded to dx's type
    size = torch.sigmoid(r).detach() if act == "silu" else torch.special.ndtr(r).detach()
    size = size + (rdx - size).abs() if act != "gelu_tanh" else (ry / r.clamp_max(-1e-9)).detach().abs() + (rdx - (ry / r.clamp_max(-1e-9)).detach()).abs()
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-30
    assert ((dx.double() - rdx).abs() <= 2 * rel * size + 1.01 * torch.finfo(dtype).eps / 2 * rdx.abs() + tiny).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows", [0, 5])
@pytest.mark.parametrize("xt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("residual", [None, torch.float32, torch.bfloat16])
def test_autocast_casts_as_linear_does_everywhere(device, rows, xt, residual):
    """On the CPU, without rows and with x already cast: F.linear's type, and the values of the cast operands."""
    g = torch.Generator().manual_seed(0)
    x, w, b = (torch.randn(s, generator=g).to(device) for s in ((rows, 64), (32, 64), (32,)))
    x, r = x.to(xt), None if residual is None else torch.randn(rows, 32, generator=g).to(device, residual)
    with torch.autocast(device, dtype=torch.bfloat16):
        y, plain = ops.linear_act(x, w, b, r, "silu"), torch.nn.functional.linear(x, w, b)
    assert y.dtype == (plain.dtype if r is None else r.dtype) and y.shape == plain.shape
    assert torch.equal(y, ops.linear_act(x.bfloat16(), w.bfloat16(), b.bfloat16(), r, "silu"))


@pytest.mark.parametrize("device", DEVICES)
def test_autocast_leaves_other_types_alone(device):
    """fp64 and whole numbers are not cast: refused on the GPU, fp64 products on the CPU."""
    x, w = torch.randn(4, 16, device=device).double(), torch.randn(8, 16, device=device).double()
    with torch.autocast(device, dtype=torch.bfloat16):
        with pytest.raises(TypeError):
            ops.linear_act(x.int(), w.int())
        with pytest.raises(TypeError):
            ops.linear_act(x, w.float())
        if device == "cuda":
            with pytest.raises(TypeError):
                ops.linear_act(x, w)
        else:
            y = ops.linear_act(x, w)
            assert y.dtype == torch.float64 and (y - x @ w.t()).abs().max() <= 1e-13


@pytest.mark.gpu
def test_more_tiles_than_a_grid_dimension_holds():
    """2^24 + 2 tiles of 64 rows, and the backward; every value is exact."""
    m = (1 << 30) + 70
    if torch.cuda.mem_get_info()[0] < 30e9:
        pytest.skip("needs 30 GB")
    x = torch.randn(m, 1, device="cuda", dtype=torch.bfloat16, generator=torch.Generator("cuda").manual_seed(0)).requires_grad_(True)
    w = torch.ones(1, 1, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = ops.linear_act(x, w, activation="relu")
    assert torch.equal(y, x.detach().clamp_min(0))
    dy = torch.zeros_like(y)
    ends = [0, 1, 1 << 29, m - 71, m - 2, m - 1]
    dy[ends] = 2.0
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    pos = (x.detach()[ends] > 0).to(dx.dtype)
    assert torch.equal(dx[ends], 2 * pos) and dx.count_nonzero() == pos.count_nonzero()
    want = (2 * pos.double() * x.detach()[ends].double()).sum()
    assert abs(dw.double().item() - want.item()) <= (2.0 ** -8 + 8 * U32) * want.abs().item() + 1e-6


@pytest.mark.gpu
def test_more_columns_than_a_grid_dimension_holds():
    """The bias gradient of 2^27 + 40 columns."""
    n = (1 << 27) + 40
    if torch.cuda.mem_get_info()[0] < 10e9:
        pytest.skip("needs 10 GB")
    x = torch.ones(1, 1, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(n, 1, device="cuda", dtype=torch.bfloat16)
    b = torch.zeros(n, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = ops.linear_act(x, w, b, activation="relu")
    dy = torch.randn(1, n, device="cuda", dtype=torch.bfloat16, generator=torch.Generator("cuda").manual_seed(0))
    (db,) = torch.autograd.grad(y, b, dy)
    assert (y == 1).all() and torch.equal(db, dy[0])
