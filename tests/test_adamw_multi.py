"""The many-tensor AdamW step (ops/adamw_multi.py, csrc/adamw_multi.hip) against the formula in 64 bits.

Tolerances.  Every sum and product of the step rounds once to fp32, by at most half a step
(2^-24 relative).  m and v are two products and a sum of them: at most 3 roundings of terms no
larger than T = b1 |m| + (1 - b1) |g| (v: all terms positive), so 4 * 2^-24 T covers them.  The
update adds a square root, a product with 1/sqrt(bc2), the sum with eps, a product with 1/bc1, the
division, the product with lr and, before all of them, half of v's own error: at most 12 * 2^-24 of
lr times the update with m replaced by T; the weight adds three roundings of its own size.
An 8-bit code may differ from the reference's where the scaled value lies within those errors
of the border that the random offset sets; then it is the neighbouring code.
"""
import math

import pytest
import torch

from scaletorch_amd import ops
from scaletorch_amd.models.gpt import GPT, GPTConfig
from scaletorch_amd.optim import MultiTensorAdamW

U = 2.0 ** -24
F8 = torch.float8_e4m3fn
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
HYPER = dict(lr=3e-3, betas=(0.9, 0.97), eps=1e-8)


def _case(sizes, device, ptype=torch.float32, gtype=torch.float32, eight=False, seed=0, offset=0, gscale=1e-3):
    """Lists as adamw_multi_ takes them; `offset`: every tensor starts that many elements into its allocation."""
    g = torch.Generator().manual_seed(seed)

    def make(shape, std, dtype=torch.float32):
        n = math.prod(shape)
        x = torch.empty(n + offset, dtype=dtype, device=device)[offset:]
        return x.copy_(torch.randn(n, generator=g).mul_(std).to(dtype)).view(shape)

    c = dict(params=[], grads=[], exp_avg=[], exp_avg_sq=[], masters=[], scales=[])
    for s in sizes:
        s = s if isinstance(s, tuple) else (s,)
        w = make(s, 0.05)
        c["params"].append(w if ptype == torch.float32 else w.to(ptype))
        c["masters"].append(None if ptype == torch.float32 else w)
        c["grads"].append(make(s, gscale, gtype))
        m, v = make(s, 0.5 * gscale), make(s, gscale).square_()
        sc = None
        if eight:
            m, v, sc = ops.adamw_pack8(m, v)
        c["exp_avg"].append(m)
        c["exp_avg_sq"].append(v)
        c["scales"].append(sc)
    return c


def _clone(c):
    return {k: [None if t is None else t.clone() for t in v] for k, v in c.items()}


def _exact(c, i, step, wd, clip, lr, betas, eps):
    """(p, m, v) after the step in 64 bits, and the bounds of their fp32 errors."""
    b1, b2 = betas
    w = c["masters"][i] if c["masters"][i] is not None else c["params"][i]
    p, g = w.double(), c["grads"][i].double() * clip
    m, v = c["exp_avg"][i], c["exp_avg_sq"][i]
    if m.dtype == F8:
        m, v = (t.double() for t in ops.adamw_unpack8(m, v, c["scales"][i]))
    m, v = m.double(), v.double()
    T = b1 * m.abs() + (1 - b1) * g.abs()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    denom = (v / (1 - b2 ** step)).sqrt() + eps
    new = p * (1 - lr * wd) - lr * (m / (1 - b1 ** step)) / denom
    dp = 12 * U * lr * (T / (1 - b1 ** step)) / denom + 3 * U * (p.abs() + new.abs())
    # decoding an 8-bit moment rounds once more, its square twice; scalars are rounded to fp32 too
    return new, m, v, 2 * dp + 1e-45, 8 * U * T + 1e-45, 10 * U * v + 1e-45


def _code_steps(q, ref):
    """How many codes q is away from ref (both e4m3, same sign)."""
    a, b = (t.view(torch.uint8).to(torch.int32) & 0x7F for t in (q, ref))
    return (a - b).abs()


SIZES = [(1,), (3,), (255,), (256,), (257,), (5, 7), (4096,), (4097,), (33, 513), ()]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("ptype,gtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                         (torch.float16, torch.float32), (torch.float32, torch.float16),
                                         (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("offset", [0, 1])
def test_step_matches_formula(device, eight, ptype, gtype, offset):
    c = _case(SIZES, device, ptype, gtype, eight, offset=offset)
    if offset and eight:
        pytest.skip("packed states are allocations of their own")
    before, step = _clone(c), 11
    wd = [0.1 if i % 2 else 0.0 for i in range(len(SIZES))]
    clip = torch.full((1,), 0.37, device=device)
    ops.adamw_multi_(**c, step=step, weight_decay=wd, clip_coef=clip, **HYPER)
    for i in range(len(SIZES)):
        p, m, v, dp, dm, dv = _exact(before, i, step, wd[i], clip.double().item(), **HYPER)
        w = c["params"][i] if ptype == torch.float32 else c["masters"][i]
        assert ((w.double() - p).abs() <= dp).all(), SIZES[i]
        if ptype != torch.float32:
            assert torch.equal(c["params"][i], w.to(ptype))
        if not eight:
            assert ((c["exp_avg"][i].double() - m).abs() <= dm).all()
            assert ((c["exp_avg_sq"][i].double() - v).abs() <= dv).all()
            continue
        for name, k, x in (("exp_avg", 0, m), ("exp_avg_sq", 1, v.sqrt())):
            blocks = torch.nn.functional.pad(x.reshape(-1), (0, -x.numel() % ops.adamw_multi.BLOCK)).view(-1, 256)
            top = blocks.abs().amax(1)
            assert torch.allclose(c["scales"][i][:, k].double(), top / 448, rtol=16 * U, atol=0)
            got = (c[name][i].float().double().reshape(-1) * c["scales"][i][:, k].double().repeat_interleave(256)[: x.numel()])
            # stochastic rounding: the value lies within one step (2^-3 of the binade, 2^-9 at least)
            # of the code's, and the root's smallest code stands for all smaller ones
            unit = top.repeat_interleave(256)[: x.numel()] / 448
            stepsize = unit * torch.exp2(torch.floor(torch.log2((x.reshape(-1).abs() / unit).clamp_min(2.0 ** -6))) - 3)
            assert ((got - x.reshape(-1)).abs() <= stepsize * (1 + 1e-5) + 1e-40).all()


@pytest.mark.gpu
@pytest.mark.parametrize("ptype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("eight", [False, True])
def test_kernel_equals_reference(ptype, eight):
    """Many tensors (several launches), three steps: the CPU reference's results."""
    sizes = [(17 * i + 1,) for i in range(101)] + [(1000, 33)]
    a = _case(sizes, "cuda", ptype, ptype, eight, seed=3)
    b = {k: [None if t is None else t.cpu() for t in v] for k, v in a.items()}
    wd = [0.01 * (i % 5) for i in range(len(sizes))]
    for step in (1, 2, 3):
        for c in (a, b):
            ops.adamw_multi_(**c, step=step, weight_decay=wd, **HYPER)
        for i in range(len(sizes)):
            w, r = ((c["masters"] if ptype == torch.bfloat16 else c["params"])[i] for c in (a, b))
            # both follow the same fp32 operations; a division or root off by one step moves the update by 2^-23
            assert (w.cpu() - r).abs().max() <= 4 * U * r.abs().max() + 16 * U * 10 * HYPER["lr"], (step, i)
            if eight:
                for name in ("exp_avg", "exp_avg_sq"):
                    off = _code_steps(a[name][i].cpu(), b[name][i])
                    assert off.max() <= 1 and (off > 0).float().mean() <= 2e-3 + 1.01 / off.numel(), (step, i, name)
                    a[name][i].copy_(b[name][i])  # a code next to the border must not carry into the next step
                a["scales"][i].copy_(b["scales"][i])
            w.copy_(r)


@pytest.mark.parametrize("device", DEVICES)
def test_rounding_is_unbiased_repeatable_and_follows_the_step(device):
    n = 256 * 400
    x = torch.linspace(0.01, 1.0, 256, device=device).repeat(400)

    def run(step):
        # beta1 = 0: m becomes the gradient, so the stored codes are the gradient's
        c = dict(params=[torch.zeros(n, device=device)], grads=[x.clone()],
                 exp_avg=[torch.zeros(n, device=device).to(F8)], exp_avg_sq=[torch.zeros(n, device=device).to(F8)],
                 scales=[torch.zeros(400, 2, device=device)])
        ops.adamw_multi_(**c, step=step, lr=1e-3, betas=(0.0, 0.0))
        return c

    a, b, other = run(5), run(5), run(6)
    for k in ("exp_avg", "exp_avg_sq"):
        assert torch.equal(a[k][0].view(torch.uint8), b[k][0].view(torch.uint8))
        assert not torch.equal(a[k][0].view(torch.uint8), other[k][0].view(torch.uint8))
    got = a["exp_avg"][0].float() * a["scales"][0][:, 0].repeat_interleave(256)
    # 400 roundings of each value, each off by less than a step d <= x / 8 with a variance of at most
    # d^2 / 4: the mean's standard deviation is at most x / 8 / 2 / 20; six of them
    mean = got.view(400, 256).mean(0)
    assert ((mean - x[:256]).abs() <= 6 * x[:256] / 320).all()
    assert (got.view(400, 256)[:, -1] == x[255]).all()  # the largest of a block is exact


@pytest.mark.parametrize("device", DEVICES)
def test_small_second_moments_move_and_never_reach_zero(device):
    n, steps = 2048, 300
    g = torch.rand(n, device=device) + 0.5
    g[::256] = 300.0  # the block's scale: most roots are far below it
    c = dict(params=[torch.zeros(n, device=device)], grads=[g], exp_avg=[torch.zeros(n, device=device).to(F8)],
             exp_avg_sq=[torch.zeros(n, device=device).to(F8)], scales=[torch.zeros(n // 256, 2, device=device)])
    for t in range(1, steps + 1):
        ops.adamw_multi_(**c, step=t, lr=1e-3, betas=(0.9, 0.999))
    _, v = ops.adamw_unpack8(c["exp_avg"][0], c["exp_avg_sq"][0], c["scales"][0])
    want = g.double() ** 2 * (1 - 0.999 ** steps)
    # rounding to nearest would hold v where one step no longer moves it; the mean follows the fp32 value.
    # A root is off by at most 12.5 % for the last step and by less for the decayed ones before it.
    small = torch.ones(n, dtype=torch.bool, device=device)
    small[::256] = False
    assert abs((v.double()[small] / want[small]).mean().item() - 1) < 0.15
    assert (c["exp_avg_sq"][0].float() > 0).all()
    # a gradient of zero: the root keeps a code and the weight stays where it can be
    tiny = torch.zeros(n, device=device)
    tiny[::256] = 1e4
    c["grads"] = [tiny]
    for t in range(steps + 1, steps + 20):
        ops.adamw_multi_(**c, step=t, lr=1e-3, betas=(0.9, 0.999))
    assert (c["exp_avg_sq"][0].float() > 0).all() and c["params"][0].abs().max() < 1.0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("eight", [False, True])
def test_non_finite_gradients_spoil_their_element_only(device, eight):
    c = _case([(600,)], device, eight=eight)
    clean = _clone(c)
    for k, bad in ((3, math.nan), (300, math.inf), (599, -math.inf)):
        c["grads"][0][k] = bad
        clean["grads"][0][k] = 0.0
    for x in (c, clean):
        for t in (1, 2):
            ops.adamw_multi_(**x, step=t, **HYPER)
    bad = ~torch.isfinite(c["params"][0])
    assert set(bad.nonzero().flatten().tolist()) == {3, 300, 599}
    # their block's scale is that of the others: the same codes wherever the bad ones did not set it
    assert torch.isfinite(c["exp_avg"][0].float()[~bad]).all()
    if not eight:
        assert torch.equal(c["params"][0][~bad], clean["params"][0][~bad])


@pytest.mark.parametrize("device", DEVICES)
def test_zero_blocks_and_empty_tensors(device):
    z = lambda *s: torch.zeros(*s, device=device)  # noqa: E731
    c = dict(params=[z(0), z(300)], grads=[z(0), z(300)], exp_avg=[z(0).to(F8), z(300).to(F8)],
             exp_avg_sq=[z(0).to(F8), z(300).to(F8)], scales=[z(0, 2), z(2, 2)])
    ops.adamw_multi_(**c, step=1, lr=1.0)
    assert all((t.float() == 0).all() for k in c for t in c[k])
    ops.adamw_multi_([], [], [], [], step=1, lr=1.0)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    def call(change, **kw):
        c = _case([(300,), (20,)], device, eight=kw.pop("eight", False))
        change(c)
        ops.adamw_multi_(**c, **{"step": 1, "lr": 1e-3, **kw})

    def put(key, i, f):
        return lambda c: c[key].__setitem__(i, f(c[key][i]))

    bad = [
        (put("params", 0, lambda t: t.bfloat16()), {}),                   # 16 bits without a master
        (put("masters", 0, lambda t: torch.zeros(300, device=device)), {}),  # fp32 with one
        (put("grads", 0, lambda t: t[:200]), {}),
        (put("grads", 0, lambda t: t.view(30, 10)), {}),
        (put("grads", 0, lambda t: t.double()), {}),
        (put("exp_avg", 1, lambda t: t.bfloat16()), {}),
        (put("exp_avg_sq", 1, lambda t: t.to(F8)), {}),
        (put("scales", 0, lambda t: None), {"eight": True}),
        (put("scales", 0, lambda t: t[:1]), {"eight": True}),
        (put("params", 0, lambda t: torch.zeros(600, device=device)[::2]), {}),
        (lambda c: c["params"].pop(), {}),
        (lambda c: c["params"].__setitem__(1, c["params"][0][:20]), {}),   # shares memory
        (lambda c: c["exp_avg_sq"].__setitem__(0, c["exp_avg"][0]), {}),
        (lambda c: c["grads"].__setitem__(0, c["params"][0]), {}),
        (lambda c: None, {"step": 0}),
        (lambda c: None, {"betas": (1.0, 0.9)}),
        (lambda c: None, {"clip_coef": torch.ones(2, device=device)}),
        (lambda c: None, {"weight_decay": [0.1]}),
    ]
    for k, (change, kw) in enumerate(bad):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call(change, **kw)
            pytest.fail(f"case {k} was not refused")
    if device == "cuda":
        with pytest.raises(RuntimeError):
            call(put("exp_avg", 0, lambda t: t.cpu()))


@pytest.mark.parametrize("device", DEVICES)
def test_shared_gradient_memory_is_allowed(device):
    """Gradients are only read: one expanded or shared buffer of them is no conflict."""
    c = _case([(64,), (64,)], device)
    c["grads"][1] = c["grads"][0]
    ops.adamw_multi_(**c, step=1, lr=1e-3)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("gtype", [torch.float32, torch.bfloat16, torch.float16])
def test_scaled_gradients_are_written_on_request(device, gtype):
    a = _case([(300,), (4099,)], device, gtype=gtype)
    b, clip = _clone(a), torch.full((1,), 0.3, device=device)
    before = _clone(a)["grads"]
    ops.adamw_multi_(**a, step=1, lr=1e-3, clip_coef=clip)
    ops.adamw_multi_(**b, step=1, lr=1e-3, clip_coef=clip, scale_grads=True)
    for i in range(2):
        assert torch.equal(a["grads"][i], before[i]) and torch.equal(a["params"][i], b["params"][i])
        assert torch.equal(b["grads"][i], (before[i].float() * clip).to(gtype))
    ops.adamw_multi_(**b, step=2, lr=1e-3, scale_grads=True)  # nothing to scale with
    b["grads"][1] = b["grads"][0]
    b["params"][1], b["exp_avg"][1], b["exp_avg_sq"][1] = (torch.zeros(300, device=device) for _ in range(3))
    with pytest.raises((ValueError, RuntimeError)):  # two tensors would scale it at once
        ops.adamw_multi_(**b, step=1, lr=1e-3, clip_coef=clip, scale_grads=True)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_optimizer_follows_torch_adamw(device, dtype):
    """32-bit moments: torch's AdamW on fp32 weights, over steps, groups and a skipped gradient."""
    torch.manual_seed(1)
    ws = [torch.randn(s, device=device) for s in ((40, 30), (30,), (7, 3))]
    mine = [torch.nn.Parameter(w.to(dtype)) for w in ws]
    theirs = [torch.nn.Parameter(w.to(dtype).float()) for w in ws]
    groups = lambda ps: [dict(params=ps[:1], weight_decay=0.1), dict(params=ps[1:], weight_decay=0.0)]  # noqa: E731
    a = MultiTensorAdamW(groups(mine), lr=1e-2, betas=(0.9, 0.95))
    b = torch.optim.AdamW(groups(theirs), lr=1e-2, betas=(0.9, 0.95))
    for k in range(6):
        for x, y in zip(mine, theirs):
            g = torch.randn(x.shape, device=device).to(dtype)
            x.grad, y.grad = g, g.float()
        if k == 2:
            mine[1].grad = theirs[1].grad = None
        a.step()
        b.step()
    for x, y in zip(mine, theirs):
        got = a.state[x].get("master", x)
        # six steps of lr times an update of at most ~3, each within some 20 roundings; the weights' own six
        assert (got - y).abs().max() <= 6 * (20 * U * 3e-2 + 4 * U * y.abs().max())
        assert dtype == torch.float32 or torch.equal(x.detach(), got.to(dtype))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["fp32", "fp8"])
def test_optimizer_state_round_trip(device, dtype, kind, tmp_path):
    torch.manual_seed(2)
    p = torch.nn.Parameter(torch.randn(300, 3, device=device).to(dtype))
    a = MultiTensorAdamW([p], lr=1e-2, state_dtype=kind)
    gs = [torch.randn(300, 3, device=device).to(dtype) for _ in range(6)]
    for g in gs[:3]:
        p.grad = g
        a.step()
    torch.save(a.state_dict(), tmp_path / "s.pt")
    saved = torch.load(tmp_path / "s.pt", weights_only=True)
    q = torch.nn.Parameter(p.detach().clone())
    b = MultiTensorAdamW([q], lr=1e-2, state_dtype=kind)
    b.load_state_dict(saved)
    other = MultiTensorAdamW([torch.nn.Parameter(p.detach().clone())], state_dtype="fp8" if kind == "fp32" else "fp32")
    other.load_state_dict(saved)
    st = other.state[other.param_groups[0]["params"][0]]
    assert st["step"] == 3 and ("scales" in st) == (kind == "fp32")
    for g in gs[3:]:
        p.grad, q.grad = g, g
        a.step()
        b.step()
    assert torch.equal(p, q)
    with pytest.raises(ValueError):
        MultiTensorAdamW([p], state_dtype="int4")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["fp32", "fp8"])
def test_gpt_configure_optimizers(device, kind):
    torch.manual_seed(0)
    m = GPT(GPTConfig(block_size=16, vocab_size=33, n_layer=2, n_head=2, n_embd=32)).to(device)
    opt = m.configure_optimizers(0.1, 1e-2, (0.9, 0.95), device, state_dtype=kind)
    assert isinstance(opt, MultiTensorAdamW)
    before = [p.detach().clone() for p in m.parameters()]
    idx = torch.randint(0, 33, (2, 16), device=device)
    for _ in range(2):
        opt.zero_grad()
        m(idx, idx)[1].backward()
        opt.step(clip_coef=torch.full((1,), 0.5, device=device))
    assert all(torch.isfinite(p).all() for p in m.parameters())
    assert sum(not torch.equal(p, q) for p, q in zip(m.parameters(), before)) >= len(before) - 1
    assert isinstance(m.configure_optimizers(0.1, 1e-2, (0.9, 0.95), device), torch.optim.AdamW)


def test_version_counter_and_closure():
    p = torch.nn.Parameter(torch.ones(4))
    opt = MultiTensorAdamW([p], lr=0.1)

    def closure():
        opt.zero_grad()
        loss = (p * p).sum()
        loss.backward()
        return loss

    assert opt.step(closure).item() == 4.0
    y = (p * p).sum()
    p.grad = torch.ones(4)
    opt.step()
    with pytest.raises(RuntimeError):  # the saved weight has changed
        y.backward()


@pytest.mark.gpu
def test_version_counter_on_gpu_and_other_stream():
    p = torch.nn.Parameter(torch.ones(1000, device="cuda"))
    opt = MultiTensorAdamW([p], lr=0.1, state_dtype="fp8")
    y = (p * p).sum()
    p.grad = torch.ones(1000, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        opt.step()
    torch.cuda.current_stream().wait_stream(st)
    assert torch.allclose(p, torch.full_like(p, 0.9), atol=1e-6)
    with pytest.raises(RuntimeError):
        y.backward()


@pytest.mark.gpu
def test_capture_is_refused():
    c = _case([(300,)], "cuda")
    ops.adamw_multi_(**c, step=1, lr=1e-3)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    err = None
    with torch.cuda.graph(g):
        x = c["params"][0] * 2
        try:
            ops.adamw_multi_(**c, step=2, lr=1e-3)
        except RuntimeError as e:
            err = e
    assert err is not None and "captured" in str(err)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(x, c["params"][0] * 2)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A tensor of more than 2^31 elements: its last ones, and the hash's upper word in the codes of the first."""
    n = (1 << 31) + 300
    free, _ = torch.cuda.mem_get_info()
    if free < 11 * n:
        pytest.skip("needs 24 GB")
    c = dict(params=[torch.ones(n, device="cuda")], grads=[torch.full((n,), 0.5, device="cuda")],
             exp_avg=[torch.zeros(n, device="cuda", dtype=F8)], exp_avg_sq=[torch.zeros(n, device="cuda", dtype=F8)],
             scales=[torch.zeros(ops.adamw_blocks(n), 2, device="cuda")])
    ops.adamw_multi_(**c, step=1, lr=0.25)
    for s in (slice(0, 300), slice(n // 2, n // 2 + 300), slice(n - 300, n)):
        assert torch.allclose(c["params"][0][s], torch.tensor(0.75, device="cuda"), atol=1e-6)
        assert (c["exp_avg"][0][s].float() == 448).all() and (c["exp_avg_sq"][0][s].float() == 448).all()
    assert (c["scales"][0][-3:] > 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["params", "grads", "exp_avg", "exp_avg_sq", "clip_coef"])
def test_forward_mode_is_refused(which):
    """The update of a tangent is not implemented; nothing is written by the refused call."""
    import torch.autograd.forward_ad as fwd

    c = _case([(300,)], "cuda")
    before, clip = _clone(c), torch.ones(1, device="cuda")
    with fwd.dual_level():
        d = {k: list(v) for k, v in c.items()}
        if which == "clip_coef":
            clip = fwd.make_dual(clip, torch.ones_like(clip))
        else:
            d[which][0] = fwd.make_dual(d[which][0], torch.ones(300, device="cuda"))
        with pytest.raises(NotImplementedError):
            ops.adamw_multi_(**d, step=1, lr=1e-3, clip_coef=clip)
    assert all(torch.equal(a, b) for k in ("params", "exp_avg", "exp_avg_sq") for a, b in zip(c[k], before[k]))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", ["params", "masters", "exp_avg", "exp_avg_sq", "scales", "grads"])
def test_a_graph_that_saved_what_a_step_writes_notices(device, which):
    """On the GPU as on the CPU: backward through an overwritten value raises."""
    eight = which == "scales"
    c = _case([(300,)], device, torch.bfloat16, torch.float32, eight)
    one = torch.ones((), device=device, requires_grad=True)
    y = (one * c[which][0]).sum()  # saves the second factor
    kw = dict(clip_coef=torch.full((1,), 0.5, device=device), scale_grads=True) if which == "grads" else {}
    ops.adamw_multi_(**c, step=1, lr=1e-3, **kw)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.gpu
@pytest.mark.parametrize("ptype,gtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("shifted", [("params", "grads", "masters"), ("grads",), ("exp_avg", "exp_avg_sq"), ("exp_avg_sq",),
                                     ("params", "grads", "masters", "exp_avg", "exp_avg_sq")])
def test_eight_bits_with_shifted_tensors(ptype, gtype, shifted):
    """Element by element where a tensor is not aligned for four at once: the same operations, the same bits."""
    a = _case(SIZES, "cuda", ptype, gtype, True, seed=7)
    b = _clone(a)
    for k in shifted:
        for i, t in enumerate(b[k]):
            if t is not None:
                b[k][i] = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].copy_(t.reshape(-1)).view(t.shape)
    for step in (1, 2):
        for c in (a, b):
            ops.adamw_multi_(**c, step=step, weight_decay=0.1, **HYPER)
    for k in a:
        for x, y in zip(a[k], b[k]):
            assert x is None or torch.equal(x.view(torch.uint8) if x.dtype == F8 else x, y.view(torch.uint8) if y.dtype == F8 else y)


@pytest.mark.gpu
def test_places_past_32_bits_enter_the_hash():
    """The codes of a tensor behind 2^32 elements of the call: rounding offsets of its place, both words of it.
    beta1 = 0, so the first moment is the gradient."""
    big, n, step = 1 << 32, 4000, 9
    if torch.cuda.mem_get_info()[0] < 40e9:
        pytest.skip("needs 40 GB")
    z = lambda m, dt=torch.float32: torch.zeros(m, dtype=dt, device="cuda")  # noqa: E731
    g = torch.randn(n, generator=torch.Generator().manual_seed(0))
    c = dict(params=[z(big), z(n)], grads=[z(big, torch.bfloat16), g.cuda()], exp_avg=[z(big, F8), z(n, F8)],
             exp_avg_sq=[z(big, F8), z(n, F8)], scales=[z(2 * ops.adamw_blocks(big)).view(-1, 2), z(2 * ops.adamw_blocks(n)).view(-1, 2)])
    ops.adamw_multi_(**c, step=step, lr=1e-3, betas=(0.0, 0.0))
    got = c["exp_avg"][1].cpu()

    def mix(x):
        x ^= x >> 16
        x = x * 0x7FEB352D & 0xFFFFFFFF
        x ^= x >> 15
        x = x * 0x846CA68B & 0xFFFFFFFF
        return x ^ x >> 16

    def codes(place):
        key = mix(step * 0x9E3779B9 & 0xFFFFFFFF)
        r16 = [mix((i & 0xFFFFFFFF) ^ mix(i >> 32 ^ key)) & 0xFFFF for i in range(place, place + n)]
        top = torch.nn.functional.pad(g, (0, -n % 256)).view(-1, 256).abs().amax(1).double().repeat_interleave(256)[:n]
        a = g.double().abs() * 448 / top
        unit = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3)  # e4m3's step there
        q = ((a / unit + torch.tensor(r16).double() / 65536).floor() * unit).clamp_max(448)
        return (q * g.sign()).float().to(F8)

    off = _code_steps(got, codes(big))
    # next to a border the fp32 scaling may fall on its other side: 2^-23 of a value over a step of 2^-3 of it
    assert off.max() <= 1 and (off > 0).sum() <= 2
    assert (_code_steps(got, codes(0)) > 0).float().mean() > 0.1  # another place, other offsets
    assert not c["exp_avg"][0].view(torch.uint8).any()
