"""Matrix product with bias, activation and residual in its epilogue (csrc/linear_act_*.hip)::

    y = act(x weight^T + bias) + residual

in one kernel, with the gradients of all four (dz = dy act'(z) and the bias gradient in one pass,
dx = dz weight, dweight = dz^T x).  ``linear`` (ops/mlp.py) is the plain product on the library
GEMM.  Reference: the biased linears, GELU and residual adds of scaletorch/models/moe.py's blocks.
Sums are fp32; y is rounded once.  What training keeps between the passes is z in x's type and, for
the products of the backward, dz in x's type: each is one rounding (2^-8 relative in bf16) of a term
of long sums, and x's type is what the matrix instructions take.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from . import _lib
from .grad import _grad_ready, accumulate_grad, take_fresh

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def _autocast_type(x: torch.Tensor) -> torch.dtype | None:
    kind = x.device.type
    return torch.get_autocast_dtype(kind) if kind in ("cuda", "cpu") and torch.is_autocast_enabled(kind) else None


def _act_ref(z: torch.Tensor, activation: str) -> torch.Tensor:
    if activation == "relu":
        return torch.relu(z)
    if activation == "gelu":
        return z * (0.5 * torch.erfc(z * -math.sqrt(0.5)))
    if activation == "gelu_tanh":  # (1 + tanh(a)) / 2 = sigmoid(2 a)
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return F.silu(z) if activation == "silu" else z


def linear_act_ref(x, weight, bias, residual, activation):
    """The same from torch operations, in fp32 (float64 for float64 inputs)."""
    f = torch.float64 if x.dtype == torch.float64 else torch.float32
    if _autocast_type(x) is not None:  # it would take F.linear back to 16 bits
        with torch.autocast(x.device.type, enabled=False):
            return linear_act_ref(x, weight, bias, residual, activation)
    z = F.linear(x.to(f), weight.to(f), None if bias is None else bias.to(f))
    y = _act_ref(z, activation)
    if residual is None:
        return y.to(x.dtype)
    return (y + residual.to(f)).to(residual.dtype)


def _weight_grad(weight, dz, x2):
    """dz^T x2 into ``main_grad`` (None), or returned.  By linear_act's own product: the backward can be captured
    into a graph, where a library product may not create its handle nor a tuner wait for its events."""
    mg = getattr(weight, "main_grad", None)
    if mg is None or not mg.is_contiguous() or mg.dtype not in (torch.float32, dz.dtype):
        return accumulate_grad(weight, _lib.ops().linear_act_dw(dz, x2))
    _lib.ops().linear_act_dw_(mg.view(weight.shape), dz, x2, not take_fresh(weight))
    _grad_ready(weight)
    return None


class _LinearActFn(torch.autograd.Function):
    """For weights with ``main_grad``; without, csrc/linear_act_ops.cpp has the same in C++."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        keep = act != 0 and any(ctx.needs_input_grad[:3])
        y, z = _lib.ops().linear_act_fwd(x, weight, bias, residual, act, keep)
        ctx.save_for_backward(x, weight, z if keep else None)
        ctx.act, ctx.bias = act, bias
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        nx, nw, nb, nr = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if nx or nw or nb:
            f32 = nb and getattr(ctx.bias, "main_grad", None) is not None
            dz, db = _lib.ops().linear_act_dz(dy, z, x.dtype, ctx.act, nb, f32)
            x2 = x.reshape(-1, x.shape[-1])
            if nx:
                dx = _lib.ops().linear_act_dx(dz, weight).view(x.shape)
            if nw:
                dw = _weight_grad(weight, dz, x2)
            db = accumulate_grad(ctx.bias, db) if nb else None
        return dx, dw, db, dy if nr else None, None


def _check(x, weight, bias, residual) -> None:
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"linear_act: weight {tuple(weight.shape)} does not take x {tuple(x.shape)}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"linear_act: bias must have shape [{weight.shape[0]}], got {tuple(bias.shape)}")
    if residual is not None and residual.shape != (*x.shape[:-1], weight.shape[0]):
        raise ValueError(f"linear_act: the residual must have y's shape {(*x.shape[:-1], weight.shape[0])}, got "
                         f"{tuple(residual.shape)}")
    if any(t is not None and t.device != x.device for t in (weight, bias, residual)):
        raise ValueError("linear_act: tensors on different devices")
    if not x.is_floating_point() or weight.dtype != x.dtype or (bias is not None and bias.dtype != x.dtype):
        raise TypeError(f"linear_act: x, weight and bias must have one floating type, got {x.dtype}, {weight.dtype}"
                        + ("" if bias is None else f", {bias.dtype}"))
    if residual is not None and residual.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"linear_act: the residual has x's type or fp32, got {residual.dtype}")


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
               residual: torch.Tensor | None = None, activation: str = "none") -> torch.Tensor:
    """``act(x weight^T + bias) + residual`` for x [..., K], weight [N, K], bias [N], residual [..., N].

    ``activation``: "none", "relu", "gelu", "gelu_tanh" or "silu".  On the GPU x, weight and bias are
    bf16 or fp16; under ``torch.autocast`` they are cast as ``F.linear`` casts them, on the CPU too.  y has the
    residual's type, which may be fp32, else x's.  Weight and bias gradients go to ``main_grad`` where it exists."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"linear_act: activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    t, native = _autocast_type(x), _lib.use_native(x)
    if t is not None:
        if native:
            _lib.check_capture(x, weight, bias, residual)  # a cast copy is no leaf: its accumulator would not be seen
        # what F.linear's cast leaves alone stays: fp64, whole numbers, other devices
        x, weight, bias = (v.to(t) if v is not None and v.is_floating_point() and v.dtype != torch.float64
                           and v.device.type == x.device.type else v for v in (x, weight, bias))
    if not native or x.numel() == 0 or weight.numel() == 0:
        _check(x, weight, bias, residual)
        return linear_act_ref(x, weight, bias, residual, activation)
    if getattr(weight, "main_grad", None) is not None or getattr(bias, "main_grad", None) is not None:
        _lib.check_capture(x, weight, bias, residual)
        return _LinearActFn.apply(x, weight, bias, residual, act)
    return _lib.ops().linear_act.default(x, weight, bias, residual, act)
