"""The norms around a block's gated residual, fused (csrc/block_norm_fwd.hip, block_norm_bwd.hip).

Between a block's output projection and the next block's first linear a decoder has::

    u = norm_post(h) * post_weight + post_bias     (or h)
    s = residual + scale * gate * u                (the new residual stream)
    y = norm_pre(s) * pre_weight + pre_bias        (what the next block reads)

``add_rms_norm`` (ops/norm.py) is the case without a norm after the block, gate and scale, in
bf16 and RMS only; ``block_norm`` has all of them, RMS and layer norms, and LayerNorm itself (no
residual).  Reference: the norms and residual adds of scaletorch/models/llama.py:320-379 and
scaletorch/models/moe.py.  Statistics, s before its rounding and every gradient sum are fp32;
y comes from the unrounded s.
"""
from __future__ import annotations

import torch

from . import _lib
from .grad import accumulate_grad

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _normalize(x: torch.Tensor, layer: bool, eps: float) -> torch.Tensor:
    if layer:
        x = x - x.mean(-1, keepdim=True)
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps)


def block_norm_ref(h, residual, layer, post_weight, post_bias, gate, scale, pre_weight, pre_bias, eps):
    """The same in elementary operations, in fp32 (float64 for float64 inputs)."""
    f = torch.float64 if h.dtype == torch.float64 else torch.float32
    u = h.to(f)
    if post_weight is not None:
        u = _normalize(u, layer, eps) * post_weight.to(f)
        if post_bias is not None:
            u = u + post_bias.to(f)
    if gate is not None:
        u = u * gate.to(f)
    s = u * scale
    if residual is not None:
        s = residual.to(f) + s
    y = None
    if pre_weight is not None:
        y = _normalize(s, layer, eps) * pre_weight.to(f)
        if pre_bias is not None:
            y = y + pre_bias.to(f)
        y = y.to(h.dtype)
    return y, s.to(h.dtype if residual is None else residual.dtype)


def _flat(*weights):
    return [None if w is None else w.contiguous() for w in weights]


class _BlockNormFn(torch.autograd.Function):
    """For weights with ``main_grad``; without, csrc/block_norm_ops.cpp has the same in C++."""

    @staticmethod
    def forward(ctx, h, residual, gate, w1, b1, w2, b2, layer, scale, eps, write_s):
        stream = h.dtype if residual is None else residual.dtype
        alone = w1 is None and gate is None and (not write_s or stream == torch.float32)
        y, s, stats = _lib.ops().block_norm_fwd(h, residual, *_flat(gate, w1, b1, w2, b2), layer, scale, eps, write_s,
                                                True)
        y = y if w2 is not None else None
        s = s if write_s else None
        # what the backward recomputes from (csrc/block_norm_bwd.hip): h and the residual, or s alone
        rows = (None, None, s if write_s else h) if alone else (h, residual, None)
        ctx.save_for_backward(*rows, stats, gate, w1, b1, w2, b2)
        ctx.meta = (layer, scale, eps, h.dtype, residual is not None, None if residual is None else residual.dtype)
        ctx.set_materialize_grads(False)
        if write_s and not any(ctx.needs_input_grad[:5]):
            ctx.mark_non_differentiable(s)
        return y, s

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, ds):
        h, residual, s, stats, gate, w1, b1, w2, b2 = ctx.saved_tensors
        layer, scale, eps, htype, has_res, rtype = ctx.meta
        if dy is None and ds is None:
            return (None,) * 11
        need = list(ctx.needs_input_grad[:7])
        gen = w1 is not None or gate is not None
        # without a norm after the block, gate or scale dh IS the residual's gradient
        one = not gen and has_res and scale == 1.0 and htype == rtype
        want = [need[0] and not one, has_res and (need[1] or (one and need[0])), *need[2:]]
        weights = (gate, w1, b1, w2, b2)
        f32 = [0, 0] + [int(w is not None and getattr(w, "main_grad", None) is not None) for w in weights]
        got = _lib.ops().block_norm_bwd(None if dy is None else dy.contiguous(), None if ds is None else ds.contiguous(),
                                        h, residual, s, stats, *_flat(*weights), layer, scale, eps,
                                        [int(w) for w in want], f32, htype)
        got = [g if w else None for g, w in zip(got, want)]
        if one and need[0]:
            got[0] = got[1]
            got[1] = got[1] if need[1] else None
        for i, w in enumerate(weights):
            if w is not None and got[2 + i] is not None:
                got[2 + i] = accumulate_grad(w, got[2 + i].view_as(w))
        return (*got, None, None, None, None)


def _check(h, residual, kind, post_weight, post_bias, gate, pre_weight, pre_bias) -> None:
    if kind not in ("rms", "layer"):
        raise ValueError(f"block_norm: kind must be 'rms' or 'layer', got {kind!r}")
    if h.dim() < 1 or h.shape[-1] < 1:
        raise ValueError(f"block_norm: h needs rows of at least one column, got {tuple(h.shape)}")
    width, small = h.shape[-1], []
    for w, what in ((gate, "gate"), (post_weight, "post_weight"), (post_bias, "post_bias"),
                    (pre_weight, "pre_weight"), (pre_bias, "pre_bias")):
        if w is None:
            continue
        if not (w.dim() == 1 and w.numel() == width or what == "gate" and w.numel() == 1 and w.dim() <= 1):
            raise ValueError(f"block_norm: {what} must have shape [{width}]"
                             + (" or one element" if what == "gate" else "") + f", got {tuple(w.shape)}")
        if w.device != h.device:
            raise ValueError(f"block_norm: {what} is on {w.device}, h on {h.device}")
        small.append(w.dtype)
    if (post_bias is not None and post_weight is None) or (pre_bias is not None and pre_weight is None):
        raise ValueError("block_norm: a bias needs its weight")
    if residual is not None:
        if residual.shape != h.shape or residual.device != h.device:
            raise ValueError(f"block_norm: the residual must be h's {tuple(h.shape)} on {h.device}, got "
                             f"{tuple(residual.shape)} on {residual.device}")
        if residual.dtype not in (h.dtype, torch.float32):
            raise TypeError(f"block_norm: the residual has h's type ({h.dtype}) or fp32, got {residual.dtype}")
    if h.dtype not in _TYPES and not (h.dtype == torch.float64 and not h.is_cuda):
        raise TypeError(f"block_norm: h must be fp32, bf16 or fp16, got {h.dtype}")
    if len(set(small)) > 1 or (small and small[0] not in (h.dtype, torch.float32)):
        raise TypeError(f"block_norm: gate and weights all have h's type ({h.dtype}) or all fp32, got {small}")


def block_norm(h: torch.Tensor, residual: torch.Tensor | None = None, *, kind: str = "rms",
               post_weight: torch.Tensor | None = None, post_bias: torch.Tensor | None = None,
               gate: torch.Tensor | None = None, scale: float = 1.0, pre_weight: torch.Tensor | None = None,
               pre_bias: torch.Tensor | None = None,
               eps: float = 1e-6) -> tuple[torch.Tensor | None, torch.Tensor]:
    """``(y, s)`` of a block's output ``h`` [..., width] and its ``residual`` (the module's formulas).

    ``kind``: "rms" or "layer", of both norms; a norm is there where its weight is.  ``gate``: one
    value, or one a column, learned.  ``residual`` may be fp32 with 16-bit h: s has its type, y has
    h's.  Without ``pre_weight`` y is None.  Rows of at most 8192 columns on the GPU.  Weight
    gradients go to ``main_grad`` where a weight has one."""
    if not _lib.use_native(h) or h.numel() == 0:
        _check(h, residual, kind, post_weight, post_bias, gate, pre_weight, pre_bias)
        return block_norm_ref(h, residual, kind == "layer", post_weight, post_bias, gate, float(scale), pre_weight,
                              pre_bias, eps)
    if kind not in ("rms", "layer"):
        raise ValueError(f"block_norm: kind must be 'rms' or 'layer', got {kind!r}")
    weights = (gate, post_weight, post_bias, pre_weight, pre_bias)
    if not any(getattr(w, "main_grad", None) is not None for w in weights):
        return _lib.ops().block_norm.default(h, residual, *weights, kind == "layer", scale, eps)
    # weights whose gradients live in an arena: the sums go there in fp32
    _check(h, residual, kind, post_weight, post_bias, gate, pre_weight, pre_bias)
    same = residual is None and post_weight is None and gate is None and scale == 1.0  # s is h itself
    _lib.check_capture(h, residual, *weights)  # the caller's: a contiguous copy is no leaf
    hc, rc = h.contiguous(), None if residual is None else residual.contiguous()
    y, s = _BlockNormFn.apply(hc, rc, *weights, kind == "layer", float(scale), eps, not same)
    return y, h if same else s
