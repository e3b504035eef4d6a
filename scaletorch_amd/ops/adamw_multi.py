"""One AdamW step over many separate tensors, moments in 32 or 8 bits (csrc/adamw_multi.hip).

The arena optimizers (optim.py) update one flat allocation per dtype; this is the step for
parameters that stay separate tensors, as ``torch.optim`` holds them (reference:
torch.optim.AdamW(fused=True), scaletorch/trainer/model_builder.py:119-134).  For every tensor::

    g = clip_coef * grad
    m = beta1 m + (1 - beta1) g            v = beta2 v + (1 - beta2) g^2
    p = p (1 - lr wd) - lr (m / (1 - beta1^t)) / (sqrt(v / (1 - beta2^t)) + eps)

in fp32.  8-bit moments (``torch.float8_e4m3fn``) hold m and the ROOT of v, each block of
``BLOCK`` consecutive elements of a tensor scaled by its largest |value| / 448 (``scales[i]``,
fp32 ``[blocks, 2]``: of m, of the root), rounded stochastically with offsets hashed from the
element's place and the step; the update itself uses the unrounded values.  A root that is not
zero is never rounded to zero.
"""
from __future__ import annotations

import math
from collections.abc import Sequence

import torch

from . import _lib

BLOCK = 256
TOP = 448.0  # largest finite value of float8_e4m3fn
_F8 = torch.float8_e4m3fn


def adamw_blocks(numel: int) -> int:
    """Blocks (rows of ``scales``) of a tensor with ``numel`` elements."""
    return -(-numel // BLOCK)


def _in_blocks(x: torch.Tensor) -> torch.Tensor:
    """Flat fp32 ``x`` as [blocks, BLOCK], the last block filled up with zeros."""
    x = x.reshape(-1).float()
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _round8(x: torch.Tensor, r16: torch.Tensor | None, root: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """[blocks, BLOCK] fp32 -> (e4m3 codes as fp32 values, scale [blocks]); ``r16``: the 16-bit
    rounding offsets, None rounds to nearest."""
    fin = torch.isfinite(x)
    ax = torch.where(fin, x.abs(), 0.0)
    top = ax.amax(1, keepdim=True)
    a = (ax * torch.where(top > 2.0 ** -100, TOP / top, 0.0)).clamp_max(TOP)
    tiny = torch.where(a < 2.0 ** -6, 2.0 ** -6, 0.0)
    off = 0x8000 if r16 is None else r16.view_as(a)
    bits = (a + tiny).view(torch.int32).to(torch.int64) + (off << 4)
    q = (bits & ~0xFFFFF).to(torch.int32).view(torch.float32) - tiny
    q = q.clamp_max(TOP)
    if root:
        q = torch.where(a > 0, q.clamp_min(2.0 ** -9), q)
    q = torch.where(fin, torch.copysign(q, x), math.nan)
    return q, (top * (1 / TOP)).squeeze(1)


def adamw_pack8(exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """fp32 moments -> (8-bit exp_avg, 8-bit root of exp_avg_sq, scales), rounded to nearest."""
    got, scales = [], []
    for x, root in ((exp_avg, False), (exp_avg_sq.sqrt(), True)):
        q, s = _round8(_in_blocks(x), None, root)
        got.append(q.view(-1)[: x.numel()].to(_F8).view(x.shape))
        scales.append(s)
    return got[0], got[1], torch.stack(scales, 1)


def adamw_unpack8(exp_avg: torch.Tensor, root: torch.Tensor, scales: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The fp32 moments (m, v) that 8-bit ones stand for."""
    m = (_in_blocks(exp_avg) * scales[:, :1]).view(-1)[: exp_avg.numel()].view(exp_avg.shape)
    r = (_in_blocks(root) * scales[:, 1:]).view(-1)[: root.numel()].view(root.shape)
    return m, r * r


def _some(ts):
    """A list for the kernel's side, which takes tensors only: empty for none, an empty tensor in a None's place."""
    if ts is None:
        return []
    if all(t is not None for t in ts):
        return ts
    none = next((t for t in ts if t is not None), None)
    return [] if none is None else [none.new_empty(0) if t is None else t for t in ts]


def _check(params, grads, exp_avg, exp_avg_sq, masters, scales, clip_coef, wd, scale_grads) -> None:
    """The checks of csrc/adamw_multi_ops.cpp, for CPU tensors."""
    n = len(params)
    if any(len(x) != n for x in (grads, exp_avg, exp_avg_sq, wd, masters, scales)):
        raise ValueError("adamw_multi: lists of different lengths")
    if clip_coef is not None and (clip_coef.numel() != 1 or clip_coef.dtype != torch.float32):
        raise ValueError("adamw_multi: clip_coef must be one fp32 value")
    spans = []
    for i, (p, g, m, v, w, s) in enumerate(zip(params, grads, exp_avg, exp_avg_sq, masters, scales)):
        for t, what in ((p, "param"), (g, "grad")):
            if t.dtype not in (torch.float32, torch.bfloat16, torch.float16):
                raise TypeError(f"adamw_multi: {what} must be fp32, bf16 or fp16, got {t.dtype}")
        if g.shape != p.shape:
            raise ValueError(f"adamw_multi: grad {i} has shape {tuple(g.shape)}, its param {tuple(p.shape)}")
        if m.dtype not in (torch.float32, _F8) or v.dtype != m.dtype:
            raise TypeError(f"adamw_multi: exp_avg and exp_avg_sq {i} must both be fp32 or both float8_e4m3fn, "
                            f"got {m.dtype} and {v.dtype}")
        if (w is not None) != (p.dtype != torch.float32):
            raise ValueError(f"adamw_multi: param {i} is " + ("16 bits wide and needs an fp32 master" if w is None
                                                              else "fp32 and takes no master"))
        if m.dtype == _F8 and (s is None or s.dtype != torch.float32):
            raise ValueError("adamw_multi: 8-bit moments need fp32 scales [blocks, 2]")
        want = [(p, "param", 1), (g, "grad", int(scale_grads)), (m, "exp_avg", 1), (v, "exp_avg_sq", 1)]
        if w is not None:
            if w.dtype != torch.float32:
                raise TypeError(f"adamw_multi: master {i} must be fp32")
            want.append((w, "master", 1))
        for t, what, written in want + ([(s, "scales", 1)] if m.dtype == _F8 else []):
            numel = 2 * adamw_blocks(p.numel()) if what == "scales" else p.numel()
            if t.device != params[0].device or not t.is_contiguous() or t.numel() != numel:
                raise ValueError(f"adamw_multi: {what} {i} must be contiguous, on {params[0].device} and have "
                                 f"{numel} elements")
            if numel:
                spans.append((t.data_ptr(), t.data_ptr() + t.nbytes, written))
    end = [0, 0]
    for lo, hi, written in sorted(spans):
        if lo < end[1] or (written and lo < end[0]):
            raise ValueError("adamw_multi: two of the tensors share memory (or one is given twice)")
        end[written] = max(end[written], hi)


def _adamw_multi_ref(params, grads, exp_avg, exp_avg_sq, masters, scales, clip_coef, wd, lr, b1, b2, eps, step,
                     scale_grads):
    from ..optim import sr_key, sr_offsets

    base = 0
    for p, g, m, v, w, s, d in zip(params, grads, exp_avg, exp_avg_sq, masters, scales, wd):
        n = p.numel()
        if not n:
            continue
        x = p if w is None else w
        gf = g.reshape(-1).float()
        if clip_coef is not None:
            gf = gf * clip_coef
            if scale_grads:
                g.copy_(gf.view_as(g))
        if m.dtype == _F8:
            mf, vf = (t.view(-1) for t in adamw_unpack8(m, v, s))
        else:
            mf, vf = m.view(-1), v.view(-1)
        mf = mf * b1 + gf * (1 - b1)
        vf = vf * b2 + gf * gf * (1 - b2)
        root = vf.sqrt()
        upd = (mf * (1 / (1 - b1 ** step))) / (root * (1 / math.sqrt(1 - b2 ** step)) + eps)
        x.copy_((x.reshape(-1) * (1 - lr * d) - upd * lr).view_as(x))
        if w is not None:
            p.copy_(w)
        nb = adamw_blocks(n)
        if m.dtype == _F8:
            r16 = sr_offsets(nb * BLOCK, sr_key(step), base * BLOCK, p.device)
            for k, (dst, val) in enumerate(((m, mf), (v, root))):
                q, top = _round8(_in_blocks(val), r16[k], bool(k))
                dst.copy_(q.view(-1)[:n].to(_F8).view_as(dst))
                s.view(-1, 2)[:, k] = top
        else:
            m.copy_(mf.view_as(m))
            v.copy_(vf.view_as(v))
        base += nb


@torch.no_grad()
def adamw_multi_(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avg: Sequence[torch.Tensor],
                 exp_avg_sq: Sequence[torch.Tensor], *, step: int, lr: float,
                 betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float | Sequence[float] = 0.0, masters: Sequence[torch.Tensor | None] | None = None,
                 scales: Sequence[torch.Tensor | None] | None = None,
                 clip_coef: torch.Tensor | None = None, scale_grads: bool = False) -> None:
    """Step number ``step`` (from 1) of AdamW over every tensor of ``params``, in place.

    ``params``: fp32, or bf16 / fp16 with an fp32 tensor in ``masters`` that is what gets updated
    (the 16-bit one is its rounded copy).  ``grads``: fp32, bf16 or fp16, of the params' shapes.
    ``exp_avg`` / ``exp_avg_sq``: fp32, or float8_e4m3fn with ``scales`` (see the module; the
    second then holds the root).  ``weight_decay``: one value, or one for each tensor.
    ``clip_coef``: a device fp32 value that every gradient is multiplied by; with ``scale_grads``
    the products are also written back, as ``torch.nn.utils.clip_grad_norm_`` leaves them (a pass
    of its own otherwise).  All tensors are contiguous, on one device, and what is written shares
    no memory with anything else; types may differ from tensor to tensor.  The
    step runs on the current stream; it takes its number from the host, so it can't be captured
    into a graph.
    """
    n = len(params)
    if step < 1:
        raise ValueError(f"adamw_multi: step counts from 1, got {step}")
    b1, b2 = betas
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
        raise ValueError(f"adamw_multi: betas must be in [0, 1), got {betas}")
    wd = [float(weight_decay)] * n if isinstance(weight_decay, (int, float)) else [float(w) for w in weight_decay]
    if not n:
        return
    if _lib.use_native(params[0]):
        _lib.ops().adamw_multi_.default(params, grads, exp_avg, exp_avg_sq, _some(masters), _some(scales), clip_coef,
                                        wd, lr, b1, b2, eps, step, scale_grads)
        return
    masters = [None] * n if masters is None else masters
    scales = [None] * n if scales is None else scales
    _check(params, grads, exp_avg, exp_avg_sq, masters, scales, clip_coef, wd, scale_grads and clip_coef is not None)
    _adamw_multi_ref(params, grads, exp_avg, exp_avg_sq, masters, scales, clip_coef, wd, lr, b1, b2, eps, step,
                     scale_grads)
