"""Linear layer with bias, activation and residual in the product's epilogue.

    y = act(x W^T + b) + r

The kernels are csrc/ops/gemm.hip; accumulation is in fp32 and the result is
rounded once.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from . import _native
from ._native import DTYPES, LinearArgs, launch, ptr, rows_of

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
RELU = ACTIVATIONS["relu"]
_PLAIN = {"none": lambda z: z, "relu": F.relu, "gelu": F.gelu, "silu": F.silu}


def linear(x, weight, bias=None, *, activation="none", residual=None):
    """``act(x @ weight.T + bias) + residual``, differentiable.

    x [..., K], weight [N, K], bias [N] and residual [..., N], all of one type
    (float32, bfloat16 or float16 on a GPU) and on one device; any strides.
    activation: "none", "relu", "gelu" (with the error function) or "silu".
    A row of x, and with gradients one of the result, is shorter than 8 MiB.
    Under autocast the operands are cast as for torch's own linear.  On the
    CPU, and while a call is traced or transformed, the formula is run by
    torch.  Runs on the current stream of x's device; can be captured into a
    graph.  Results do not depend on the run: sums have a fixed order.
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation {activation!r}: one of {', '.join(ACTIVATIONS)}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} does not fit weight {tuple(weight.shape)}")
    n, k = weight.shape
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"bias {tuple(bias.shape)}, wanted ({n},)")
    if residual is not None and residual.shape != x.shape[:-1] + (n,):
        raise ValueError(f"residual {tuple(residual.shape)}, wanted {tuple(x.shape[:-1]) + (n,)}")
    if _native.autocast(x.device):
        dtype = torch.get_autocast_dtype(x.device.type)
        x, weight, bias, residual = (
            t if t is None or t.dtype == torch.float64 else t.to(dtype)
            for t in (x, weight, bias, residual))
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is not None and t.dtype != x.dtype:
            raise TypeError(f"{name} is {t.dtype}, x {x.dtype}")
    _native.same_device("x weight bias residual", x, weight, bias, residual)
    if not _native.on_gpu(x, weight, bias, residual):
        return formula(x, weight, bias, residual, activation)
    if x.dtype not in DTYPES:
        raise TypeError(f"linear on a GPU takes float32, bfloat16 or float16, not {x.dtype}")
    if k * x.element_size() >= 1 << 23:
        raise ValueError(f"linear over {k} inputs: a row must be shorter than 8 MiB")
    if x.numel() == 0 or weight.numel() == 0:
        return formula(x, weight, bias, residual, activation)
    if _native.needs_grad(x, weight, bias, residual):
        if n * x.element_size() >= 1 << 23:
            raise ValueError(f"linear with gradients over {n} outputs: a row must be shorter "
                             "than 8 MiB")
        return _Linear.apply(x, weight, bias, residual, activation)
    return _forward(x, weight, bias, residual, ACTIVATIONS[activation], False)[0]


def formula(x, weight, bias, residual, activation):
    """The same by torch's own operations, for any type and device."""
    y = _PLAIN[activation](F.linear(x, weight, bias))
    return y if residual is None else y + residual


def _launch(a, device):
    """Runs a call with the workspace that it takes."""
    size = _native.entry("linear_work")(a)
    if size:
        if size < 0:
            raise ValueError("linear: an axis is too long" if size == -2
                             else "linear: vgpu_ops_linear refused the arguments")
        work = torch.empty(size, dtype=torch.uint8, device=device)
        a.work, a.work_bytes = work.data_ptr(), size
    launch("linear", device, a)


def _matrix(t, k):
    return t if t.dim() == 2 else t.reshape(-1, k)


def _forward(x, weight, bias, residual, act, keep):
    """y, and what backward needs for the activation's slope: the value before
    it, or, where y tells as much (relu without a residual), y itself."""
    n, k = weight.shape
    x2 = _matrix(x, k)
    shape = (x2.shape[0], n) if x.dim() == 2 else x.shape[:-1] + (n,)
    y = x.new_empty(shape)
    z = None
    if keep and act and not (act == RELU and residual is None):
        # rounded like y: the slope is taken where a separate layer would
        # have stored its input
        z = x.new_empty(shape)
    if bias is not None and n > 1 and bias.stride(0) != 1:
        bias = bias.contiguous()
    r2 = None if residual is None else rows_of(residual, n)
    _launch(LinearArgs(
        x2.data_ptr(), weight.data_ptr(), ptr(bias), ptr(r2), None, y.data_ptr(), ptr(z), None,
        None, None, None, x2.shape[0], n, k, *x2.stride(), *weight.stride(),
        0 if r2 is None else r2.stride(0), 0, 0, DTYPES[x.dtype], act), x.device)
    return y, (y if z is None else z) if act else None


def _formula_gradients(dy, x, weight, z, needed):
    """Those of an activation whose slope is 0 or 1, by torch's operations.  x
    and weight are there where a gradient takes them."""
    dz = dy if z is None else torch.where(z <= 0, 0.0, dy)
    flat = dz.reshape(-1, dz.shape[-1])
    return (dz @ weight if needed[0] else None,
            flat.t() @ x.reshape(-1, x.shape[-1]) if needed[1] else None,
            flat.sum(0) if needed[2] else None)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        y, z = _forward(x, weight, bias, residual, ACTIVATIONS[activation], True)
        # what no gradient takes may be changed before the backward pass, as
        # with torch's own; the derivative of a bent slope takes x and weight
        bent = activation not in ("none", "relu")
        need_x, need_w = ctx.needs_input_grad[:2]
        ctx.activation, ctx.k = activation, x.shape[-1]
        ctx.bias = (bias, bias._version) if bent and bias is not None else None
        ctx.save_for_backward(x if need_w or bent else None, weight if need_x or bent else None,
                              None if z is None else z.view_as(y))
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        needed = ctx.needs_input_grad[:3]
        dr = dy if ctx.needs_input_grad[3] else None
        if _native.formula_backward():
            return (*_formula_gradients(ctx, x, weight, z, needed, dy), dr, None)
        n, k = dy.shape[-1], ctx.k
        dy2 = rows_of(dy.resolve_neg(), n)
        dx = dy.new_empty(dy.shape[:-1] + (k,)) if needed[0] else None
        dw = dy.new_empty((n, k)) if needed[1] else None
        db = dy.new_empty(n) if needed[2] else None
        if any(needed):
            x2 = _matrix(x, k) if needed[1] else None
            _launch(LinearArgs(
                ptr(x2), ptr(weight) if needed[0] else None, None, None, dy2.data_ptr(), None, ptr(z),
                ptr(dx), ptr(dw), ptr(db), None, dy2.shape[0], n, k,
                *((0, 0) if x2 is None else x2.stride()),
                *(weight.stride() if needed[0] else (0, 0)), 0, dy2.stride(0), 0, DTYPES[dy.dtype],
                ACTIVATIONS[ctx.activation]), dy.device)
        return dx, dw, db, dr, None


def _formula_gradients(ctx, x, weight, z, needed, dy):
    """The same by torch's operations."""
    if ctx.activation in ("none", "relu"):
        dz = dy if z is None else torch.where(z <= 0, 0.0, dy)
        rows = dz.reshape(-1, dz.shape[-1])
        return ((rows @ weight).reshape(dy.shape[:-1] + (ctx.k,)) if needed[0] else None,
                rows.t() @ _matrix(x, ctx.k) if needed[1] else None,
                rows.sum(0) if needed[2] else None)
    bias, version = ctx.bias or (None, 0)
    if bias is not None and bias._version != version:
        raise RuntimeError("linear: the bias has been changed in place; the formula's gradient of "
                           f"{ctx.activation} needs it as it was")
    return _native.gradients_of(lambda x, w, b: formula(x, w, b, None, ctx.activation),
                                (x, weight, bias), needed, dy)
