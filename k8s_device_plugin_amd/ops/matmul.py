"""Linear layer with bias, activation and residual in the product's epilogue.

    y = act(x W^T + b) + r

The kernels are csrc/ops/gemm.hip; accumulation is in fp32 and the result is
rounded once.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache

import torch
import torch.nn.functional as F

from . import _native
from ._native import DTYPES, GemmArgs, SlopeArgs, launch, ptr, rows_of

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
_PLAIN = {"none": lambda z: z, "relu": F.relu, "gelu": F.gelu, "silu": F.silu}


def linear(x, weight, bias=None, *, activation="none", residual=None):
    """``act(x @ weight.T + bias) + residual``, differentiable.

    x [..., K], weight [N, K], bias [N] and residual [..., N], all of one type
    (float32, bfloat16 or float16 on a GPU) and on one device; any strides.
    activation: "none", "relu", "gelu" (with the error function) or "silu".
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
    if torch.is_autocast_enabled(x.device.type):
        dtype = torch.get_autocast_dtype(x.device.type)
        x, weight, bias, residual = (
            t if t is None or t.dtype == torch.float64 else t.to(dtype)
            for t in (x, weight, bias, residual))
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is not None and t.dtype != x.dtype:
            raise TypeError(f"{name} is {t.dtype}, x {x.dtype}")
    _native.same_device(x=x, weight=weight, bias=bias, residual=residual)
    if not _native.on_gpu(x, weight, bias, residual):
        return formula(x, weight, bias, residual, activation)
    if x.dtype not in DTYPES:
        raise TypeError(f"linear on a GPU takes float32, bfloat16 or float16, not {x.dtype}")
    if k * x.element_size() >= 1 << 23:
        raise ValueError(f"linear over {k} inputs: a row must be shorter than 8 MiB")
    if x.numel() == 0 or weight.numel() == 0:
        return formula(x, weight, bias, residual, activation)
    if _native.needs_grad(x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, residual, activation)
    return _forward(x, weight, bias, residual, ACTIVATIONS[activation], False)[0]


def formula(x, weight, bias, residual, activation):
    """The same by torch's own operations, for any type and device."""
    y = _PLAIN[activation](F.linear(x, weight, bias))
    return y if residual is None else y + residual


@lru_cache(maxsize=4096)
def _plan(m, n, k, dtype, a_kc, b_kc, bare):
    plan, splits, rows = ctypes.c_int32(), ctypes.c_int32(), ctypes.c_int64()
    _native.library().vgpu_ops_gemm_plan(m, n, k, dtype, a_kc, b_kc, bare, ctypes.byref(plan),
                                         ctypes.byref(splits), ctypes.byref(rows))
    return plan.value, splits.value, rows.value


def _operand(t, any_axis=True):
    """A matrix [rows, k] as the kernel reads it: (tensor, ld, k contiguous,
    bytes that may be read, k).  Loads are 16 bytes wide, so rows that do not
    start on 16 bytes, or that end inside 16, are laid out anew with zeros
    behind; so is a matrix that is contiguous along neither axis, or not along
    k where any_axis is false."""
    rows, k = t.shape
    s0, s1 = t.stride()
    size = t.element_size()
    if t.data_ptr() % 16 == 0:
        if rows == 1 and s1 == 1:
            s0 = k
        if s1 == 1 and k * size % 16 == 0 and s0 * size % 16 == 0 and s0 * size < 1 << 23:
            return t, s0, 1, ((rows - 1) * s0 + k) * size, k
        if any_axis and s0 == 1 and s1 >= rows and s1 * size % 16 == 0 and s1 * size < 1 << 23:
            # the last row's last load is whole: its 16 bytes are one line's
            return t, s1, 0, -(-((k - 1) * s1 + rows) * size // 16) * 16, k
    wide = -(-k * size // 16) * 16 // size
    if wide * size >= 1 << 23:
        raise ValueError(f"linear: {k} values to sum over, the most is {(1 << 23) // size - 8}")
    out = torch.empty((rows, wide), dtype=t.dtype, device=t.device)
    launch("repack", t.device, t.data_ptr(), s0, s1, rows, k, out.data_ptr(), wide,
           DTYPES[t.dtype])
    return out, wide, 1, rows * wide * size, wide


def _gemm(a, b, out, bias=None, residual=None, act=0, z=None):
    """out [m, n] = act(a [m, k] b [n, k]^T + bias) + residual."""
    m, n = out.shape
    dtype = DTYPES[out.dtype]
    # few rows are read with k contiguous, but for the short sums of a
    # weight's gradient
    a, lda, a_kc, a_extent, ka = _operand(a, m > 32 or a.shape[1] <= 32)
    b, ldb, b_kc, b_extent, kb = _operand(b)
    # a k that one side pads with zeros ends beyond the other's extent, which
    # reads as zeros there too
    k = max(ka, kb)
    bare = bias is None and residual is None and z is None and not act
    plan, splits, rows = _plan(m, n, k, dtype, a_kc, b_kc, bare)
    if rows < m:
        _gemm(a[rows:], b, out[rows:], bias, None if residual is None else residual[rows:], act,
              None if z is None else z[rows:])
        m = rows
    work = (torch.empty(splits * m * n, dtype=torch.float32, device=out.device)
            if splits > 1 else None)
    launch("gemm", out.device, GemmArgs(
        a.data_ptr(), b.data_ptr(), lda, ldb, a_extent, b_extent, m, n, k, ptr(bias),
        ptr(residual), residual.stride(0) if residual is not None else 0, out.data_ptr(),
        out.stride(0), ptr(z), z.stride(0) if z is not None else 0, ptr(work),
        dtype, a_kc, b_kc, act, plan, splits))


def _forward(x, weight, bias, residual, act, keep):
    """y, and what backward needs for the activation's slope: the value before
    it, or, where y tells as much (relu without a residual), y itself."""
    n, k = weight.shape
    y = torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=x.device)
    y2 = y.view(-1, n)
    z = None
    if keep and act and not (act == ACTIVATIONS["relu"] and residual is None):
        # rounded like y: the slope is taken where a separate layer would
        # have stored its input
        z = torch.empty_like(y2)
    if bias is not None and n > 1 and bias.stride(0) != 1:
        bias = bias.contiguous()
    _gemm(x.reshape(-1, k), weight, y2, bias,
          None if residual is None else rows_of(residual, n), act, z)
    return y, (y2 if z is None else z) if act else None


def _slope(dy, z, act, want_dz, want_db, dtype):
    """dz = dy act'(z) (rows padded with zeros to 16 bytes) and its columns'
    sums."""
    m, n = dy.shape
    code = DTYPES[dtype]
    lanes = 16 // dy.element_size()
    wide = -(-n // lanes) * lanes
    dz = torch.empty((m, wide), dtype=dtype, device=dy.device) if want_dz else None
    db = part = None
    parts = _native.plan("slope_parts", m, n, code)
    if want_db:
        db = torch.empty(n, dtype=dtype, device=dy.device)
        part = torch.empty(parts * n, dtype=torch.float32, device=dy.device)
    launch("slope", dy.device, SlopeArgs(
        dy.data_ptr(), ptr(z), ptr(dz), ptr(db), ptr(part), dy.stride(0),
        z.stride(0) if z is not None else 0, wide, m, n, code, act, parts))
    return dz, db


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        y, z = _forward(x, weight, bias, residual, ACTIVATIONS[activation], True)
        ctx.activation = activation
        ctx.save_for_backward(x, weight, bias, None if z is None else z.view_as(y))
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, bias, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dr = dy if need_r else None
        if torch.is_grad_enabled():
            found = _native.gradients_of(
                lambda x, w, b: formula(x, w, b, None, ctx.activation), (x, weight, bias),
                (need_x, need_w, need_b), dy)
            return (*found, dr, None)
        n, k = weight.shape
        act = ACTIVATIONS[ctx.activation]
        dz = rows_of(dy, n)
        db = None
        # the products read 16 bytes at a time: rows of dy that do not allow
        # it are copied along with the slope
        size = dy.element_size()
        loose = n * size % 16 or dz.stride(0) * size % 16 or dz.data_ptr() % 16
        products = need_x or need_w
        if need_b or (products and (act or loose)):
            copy = products and bool(act or loose)
            out, db = _slope(dz, None if z is None else z.view(-1, n), act, copy, need_b, dy.dtype)
            dz = out if copy else dz
        dx = dw = None
        if need_x:
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            _gemm(dz, weight.t(), dx.view(-1, k))
        if need_w:
            dw = torch.empty((n, k), dtype=x.dtype, device=x.device)
            _gemm(dz[:, :n].t(), x.reshape(-1, k).t(), dw)
        return dx, dw, db, dr, None
