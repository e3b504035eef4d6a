"""GPT blocks through the fused operators (linear_act, block_norm) and the many-tensor AdamW, together."""
import pytest
import torch

from scaletorch_amd.models.gpt import GPT, GPTConfig
from scaletorch_amd.optim import MultiTensorAdamW

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
VARIANTS = [dict(), dict(bias=False), dict(post_norm=True), dict(residual_gate=True, gate_init=0.3),
            dict(post_norm=True, residual_gate=True, gate_init=0.5, residual_scale=0.25), dict(residual_scale=0.5)]


def _model(fused, n_embd=128, **kw):
    torch.manual_seed(0)
    cfg = dict(block_size=64, vocab_size=97, n_layer=2, n_head=2, n_embd=n_embd)
    return GPT(GPTConfig(**{**cfg, **kw}, fused_ops=fused))


def _grads(m, idx, cast=None):
    if cast is None:
        loss = m(idx, idx)[1]
    else:
        with torch.autocast("cuda", dtype=cast):
            loss = m(idx, idx)[1]
    loss.backward()
    return loss.detach().double(), {n: p.grad.double() for n, p in m.named_parameters()}


def _off(a, b):
    return {n: ((a[n] - b[n]).norm() / b[n].norm().clamp_min(1e-12)).item() for n in b}


@pytest.mark.parametrize("kw", VARIANTS)
def test_fused_block_is_the_same_model_cpu(kw):
    """fp32 on the CPU: the same parameters, values and gradients (other orders of fp32 sums)."""
    a, b = _model(False, **kw), _model(True, **kw)
    assert [n for n, _ in a.named_parameters()] == [n for n, _ in b.named_parameters()]
    idx = torch.randint(0, 97, (3, 40))
    (la, ga), (lb, gb) = _grads(a, idx), _grads(b, idx)
    # some 30 fp32 operations deep, sums of up to 512 terms: 1e-5 is 170 roundings of 2^-24
    assert abs(la - lb) <= 1e-5 * la and max(_off(gb, ga).values()) <= 1e-4


def test_default_model_has_no_new_parameters():
    names = [n for n, _ in _model(False).named_parameters()]
    assert not any("join" in n for n in names)
    extra = [n for n, _ in _model(False, post_norm=True, residual_gate=True).named_parameters() if n not in names]
    assert len(extra) == 2 * 2 * 3  # a weight, a bias and a gate for both branches of two layers


@pytest.mark.gpu
@pytest.mark.parametrize("kw", VARIANTS)
@pytest.mark.parametrize("mode", ["bf16", "fp16", "autocast"])
def test_fused_block_gpu(kw, mode):
    """Against the model in fp32: no further off than the unfused one of the same types, which rounds
    at more places, would be by twice its own error (two independent sets of roundings)."""
    idx = torch.randint(0, 97, (3, 64), device="cuda")
    _, exact = _grads(_model(False, **kw).cuda(), idx)
    off = {}
    for fused in (False, True):
        m = _model(fused, **kw).cuda()
        if mode != "autocast":
            m = m.to(torch.bfloat16 if mode == "bf16" else torch.float16)
        _, g = _grads(m, idx, torch.bfloat16 if mode == "autocast" else None)
        off[fused] = _off(g, exact)
    floor = 2.0 ** -8 if mode != "fp16" else 2.0 ** -10
    for n, e in off[True].items():
        assert e <= 2 * off[False][n] + floor, (n, e, off[False][n])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["fp32", "fp8"])
def test_training_steps_together(device, kind):
    """Fused blocks, their gradients and the optimizer over several steps, captured forward and
    backward not needed: everything finite, every parameter moves, and the first step is AdamW's."""
    m = _model(True, post_norm=True, residual_gate=True).to(device)
    if device == "cuda":
        m = m.bfloat16()
    opt = m.configure_optimizers(0.1, 1e-3, (0.9, 0.95), device, state_dtype=kind)
    assert isinstance(opt, MultiTensorAdamW)
    first = {n: p.detach().clone() for n, p in m.named_parameters()}
    for step in range(4):
        idx = torch.randint(0, 97, (2, 64), device=device, generator=torch.Generator(device).manual_seed(step))
        opt.zero_grad()
        m(idx, idx)[1].backward()
        if step == 0:
            grads = {n: p.grad.clone() for n, p in m.named_parameters()}
        opt.step()
        if step == 0:
            for n, p in m.named_parameters():
                w = opt.state[p].get("master", p)
                wd = 0.1 if p.dim() >= 2 else 0.0
                g = grads[n].double()
                want = first[n].double() * (1 - 1e-3 * wd) - 1e-3 * g / (g.abs() + 1e-8)  # m / sqrt(v) of a first step
                # fp32 roundings of the weight and of some ten operations of an update of 1e-3
                assert ((w.double() - want).abs() <= 4 * 2.0 ** -24 * first[n].double().abs() + 20 * 2.0 ** -24 * 1e-3 + 1e-12).all(), n
    assert all(torch.isfinite(p).all() for p in m.parameters())
    assert all(not torch.equal(p, first[n]) for n, p in m.named_parameters() if n != "transformer.wpe.weight")


def test_fused_weights_are_waited_for():
    """The arena's bucket waits cover what the fused blocks read without calling its modules."""
    from scaletorch_amd.parallel.data_parallel import DataParallel

    idx = torch.randint(0, 97, (2, 16))
    left = {}
    for fused in (False, True):
        dp = DataParallel(_model(fused, post_norm=True, residual_gate=True), expose_grads=True)
        left[fused] = dp.uncovered_params(lambda: dp(idx, idx))
    assert left[True] == left[False]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["fp32", "fp8"])
def test_in_data_parallel_arenas(device, kind):
    """Parameters in arenas (views, fp32 main_grad): the gradients of the bare model and a step."""
    from scaletorch_amd.parallel.data_parallel import DataParallel

    idx = torch.randint(0, 97, (2, 32), device=device)
    dt = torch.bfloat16 if device == "cuda" else torch.float32
    bare, inner = (_model(True, post_norm=True, residual_gate=True).to(device, dt) for _ in range(2))
    _, want = _grads(bare, idx)
    dp = DataParallel(inner, bucket_size=1 << 16, expose_grads=True)
    opt = inner.configure_optimizers(0.1, 1e-3, (0.9, 0.95), device, state_dtype=kind)
    for _ in range(2):
        dp.zero_grad()
        dp(idx, idx)[1].backward()
        got = {n: p.grad.double() for n, p in inner.named_parameters()}
        # the arena keeps fp32 sums where the bare model rounds them to bf16 once
        assert max(_off(got, want).values()) <= (2.0 ** -7 if device == "cuda" else 1e-5)
    before = [p.detach().clone() for p in inner.parameters()]
    opt.step()
    assert all(torch.isfinite(p).all() for p in inner.parameters())
    # the masters move: a step of 1e-3 is below half a bf16 step of a weight of one
    now = [opt.state[p].get("master", p) for p in inner.parameters()]
    assert all(not torch.equal(p, q.float()) for (n, _), p, q in zip(inner.named_parameters(), now, before) if "wpe" not in n)


def test_mingpt_example_runs_fused_with_8_bit_states(tmp_path):
    import subprocess
    import sys

    import yaml
    root = __import__("os").path.dirname(__import__("os").path.dirname(__file__))
    cfg = yaml.safe_load(open(f"{root}/examples/mingpt/gpt2_train_cfg.yaml"))
    cfg["gpt_config"] |= dict(n_layer=2, n_head=2, n_embd=32, fused_ops=True, post_norm=True, residual_gate=True)
    cfg["gpt_config"].pop("model_type", None)
    cfg["data_config"] |= dict(block_size=32, truncate=0.2)
    cfg["trainer_config"] |= dict(batch_size=4, max_epochs=1, data_loader_workers=0)
    cfg["optimizer_config"]["state_dtype"] = "fp8"
    (tmp_path / "c.yaml").write_text(yaml.safe_dump(cfg))
    out = subprocess.run([sys.executable, f"{root}/examples/mingpt/main.py", "--cpu", "--max_iters", "3", "--config",
                          str(tmp_path / "c.yaml"), "--snapshot_path", str(tmp_path / "s.pt")], capture_output=True,
                         text=True, timeout=300, cwd=root)
    assert out.returncode == 0, out.stderr[-2000:]
    assert "final train loss" in out.stdout and "nan" not in out.stdout


@pytest.mark.gpu
def test_generation_one_token_at_a_time():
    """Few rows: the streaming product kernel, against the unfused model's choices at fp32 logits."""
    a, b = (_model(f).cuda().bfloat16().eval() for f in (False, True))
    idx = torch.randint(0, 97, (1, 1), device="cuda")
    with torch.no_grad():
        la, lb = a(idx)[0].float(), b(idx)[0].float()
    assert ((la - lb).norm() / la.norm()).item() <= 4 * 2.0 ** -8  # a few bf16 roundings apart
    out = b.generate(idx, 8, do_sample=False)
    assert out.shape == (1, 9) and (out < 97).all()


@pytest.mark.parametrize("kw", VARIANTS)
@pytest.mark.parametrize("mode", ["train", "eval with dropout on", "rate changed"])
def test_dropout_comes_before_the_residual(kw, mode):
    """fp32 on the CPU, the same random numbers: dropout falls on the branch's output, never on the residual stream,
    whichever way it was switched on."""
    out = {}
    for fused in (False, True):
        m = _model(fused, dropout=0.0 if mode == "rate changed" else 0.5, **kw)
        m.train(mode == "train")
        for d in m.modules():
            if isinstance(d, torch.nn.Dropout):
                d.train()
                d.p = 0.5
        torch.manual_seed(3)
        out[fused] = m(torch.randint(0, 97, (2, 24), generator=torch.Generator().manual_seed(1)))[0]
    # other orders of the same fp32 sums, as above
    assert (out[True] - out[False]).norm() <= 1e-5 * out[False].norm()


@pytest.mark.gpu
def test_an_fp32_model_on_the_gpu_says_that_it_runs_unfused():
    import warnings

    idx = torch.randint(0, 97, (2, 32), device="cuda")
    with torch.no_grad():
        want = _model(False).cuda()(idx)[0]
        with pytest.warns(UserWarning, match="unfused"):
            got = _model(True).cuda()(idx)[0]
        assert torch.equal(got, want)
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            _model(True).cuda().bfloat16()(idx)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", VARIANTS)
def test_arenas_under_autocast(kw):
    """fp32 parameters in arenas, 16-bit products: the gradients of the bare model, over two accumulated passes."""
    from scaletorch_amd.parallel.data_parallel import DataParallel

    idx = torch.randint(0, 97, (2, 64), device="cuda")
    bare, inner = (_model(True, **kw).cuda() for _ in range(2))
    _, want = _grads(bare, idx, torch.bfloat16)
    dp = DataParallel(inner, bucket_size=1 << 16, expose_grads=True)
    for _ in range(2):
        dp.zero_grad()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = dp(idx, idx)[1]
        loss.backward()
        got = {n: p.grad.double() for n, p in inner.named_parameters()}
        # the same products; only fp32 sums of the norms' weights may be added up in another order
        assert max(_off(got, want).values()) <= 1e-5
