"""Layer norm over groups of neighbouring values.

    y = (x - mean) / sqrt(var + eps) * weight + bias

The kernels are csrc/ops/norm.hip; statistics and the weight's gradient are
summed in fp32.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from . import _native
from ._native import DTYPES, NormArgs, launch, ptr, rows_of

WIDEST = 32768  # values of a group: what one workgroup's registers hold


def layer_norm(x, weight=None, bias=None, *, groups=1, eps=1e-5):
    """Normalises each of ``groups`` equal parts of x's last axis, then scales
    and shifts by weight and bias [x.shape[-1]]; differentiable.

    ``groups=1`` is layer norm; more is group norm of rows that have no extent
    beside their channels.  x: float32, bfloat16 or float16 on a GPU, any
    strides, groups of at most 32768 values; weight and bias: x's type or
    float32, both the same.  Under autocast x is normalised in float32, as by
    torch's own.  On the CPU, and while a call is traced or transformed, the
    formula is run by torch.  Runs on the current stream of x's device; can be
    captured into a graph.  Results do not depend on the run.
    """
    if x.dim() < 1 or groups < 1 or x.shape[-1] == 0 or x.shape[-1] % groups:
        raise ValueError(f"x {tuple(x.shape)} does not split into {groups} groups")
    width = x.shape[-1]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.shape != (width,):
            raise ValueError(f"{name} {tuple(t.shape)}, wanted ({width},)")
    if _native.autocast(x.device) and x.dtype != torch.float64:
        x, weight, bias = (t if t is None else t.float() for t in (x, weight, bias))
    kind = _kind(x, weight, bias)
    if kind not in (x.dtype, torch.float32) or (bias is not None and bias.dtype != kind):
        kinds = {t.dtype for t in (weight, bias) if t is not None}
        raise TypeError(f"weight and bias are {kinds}: wanted both {x.dtype} or both float32")
    _native.same_device("x weight bias", x, weight, bias)
    if not _native.on_gpu(x, weight, bias):
        return _plain(x, weight, bias, groups, eps)
    if x.dtype not in DTYPES:
        raise TypeError(f"layer_norm on a GPU takes float32, bfloat16 or float16, not {x.dtype}")
    if width // groups > WIDEST or groups > 65535:
        raise ValueError(f"layer_norm: groups of at most {WIDEST} values, at most 65535 groups")
    if x.numel() == 0:
        return _plain(x, weight, bias, groups, eps)
    if _native.needs_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, groups, eps)
    return _forward(x, weight, bias, groups, eps, False)[0]


def _plain(x, weight, bias, groups, eps):
    kind = x.dtype if x.dtype == torch.float64 else torch.float32
    y = F.layer_norm(x.to(kind).unflatten(-1, (groups, -1)), (x.shape[-1] // groups,), eps=eps)
    y = y.flatten(-2)
    if weight is not None:
        y = y * weight
    if bias is not None:
        y = y + bias
    return y.to(x.dtype)


def _vector(t):
    return t if t is None or t.stride(0) == 1 or t.numel() == 1 else t.contiguous()


def _kind(x, weight, bias):
    return weight.dtype if weight is not None else x.dtype if bias is None else bias.dtype


def _forward(x, weight, bias, groups, eps, keep):
    width = x.shape[-1]
    x2 = rows_of(x, width)
    rows = x2.shape[0]
    y = x.new_empty(x.shape)
    stats = (torch.empty((2, rows * groups), dtype=torch.float32, device=x.device)
             if keep else None)
    weight, bias = _vector(weight), _vector(bias)
    kind = _kind(x, weight, bias)
    at = ptr(stats)
    launch("norm", x.device, NormArgs(
        x2.data_ptr(), ptr(weight), ptr(bias), None, y.data_ptr(), None, None, None,
        at, at and at + 4 * rows * groups, None, x2.stride(0), width, 0, 0, rows, groups,
        width // groups, DTYPES[x.dtype], DTYPES[kind], 0, eps))
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps):
        y, stats = _forward(x, weight, bias, groups, eps, True)
        ctx.groups, ctx.eps, ctx.kind = groups, eps, _kind(x, weight, bias)
        ctx.save_for_backward(x, weight, stats)  # no gradient takes the bias
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        groups, kind = ctx.groups, ctx.kind
        width = x.shape[-1]
        if _native.formula_backward():
            bias = x.new_zeros(width, dtype=kind).requires_grad_() if need_b else None
            return (*_native.gradients_of(
                lambda x, w, b: _plain(x, w, b, groups, ctx.eps), (x, weight, bias),
                (need_x, need_w, need_b), dy), None, None)
        x2, dy2 = rows_of(x, width), rows_of(dy.resolve_neg(), width)
        rows, d = x2.shape[0], width // groups
        dx = x.new_empty(x.shape) if need_x else None
        dw = x.new_empty(width, dtype=kind) if need_w else None
        db = x.new_empty(width, dtype=kind) if need_b else None
        parts = _native.plan("norm_parts", rows, groups, d)
        part = (torch.empty(2 * parts * width, dtype=torch.float32, device=x.device)
                if parts > 1 and (need_w or need_b) else None)
        weight = _vector(weight)
        launch("norm", x.device, NormArgs(
            x2.data_ptr(), ptr(weight), None, dy2.data_ptr(), None, ptr(dx), ptr(dw), ptr(db),
            stats.data_ptr(), stats.data_ptr() + 4 * rows * groups, ptr(part), x2.stride(0), 0,
            dy2.stride(0), width, rows, groups, d, DTYPES[x.dtype], DTYPES[kind], parts, ctx.eps))
        return dx, dw, db, None, None
