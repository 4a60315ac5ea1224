"""Distillation from a teacher's top logits; with one slot, cross entropy.

    p = softmax(teacher / T) over a row's slots
    q = softmax(logits / T) over the vocabulary
    loss = T^2 sum_k p_k (log p_k - log q[index_k])

The kernels are csrc/ops/distill.hip; the softmax's maximum and sum are held
in fp32.
"""
from __future__ import annotations

import torch

from . import _native
from ._native import DTYPES, DistillArgs, launch, ptr, rows_of

REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
MOST_SLOTS = 1024


def distill_loss(logits, index, teacher=None, *, temperature=1.0, reduction="mean"):
    """The loss of ``logits`` [..., V] against a teacher whose top classes
    are ``index`` [..., K] (int32 or int64) with logits ``teacher`` [..., K].

    A slot with a negative index, or a teacher's logit of -inf, is empty; a
    row whose slots are all empty has loss 0 and gradient 0.  A class that is
    named twice counts with both masses.  An index of V or more makes the
    row's loss and gradient NaN.  Without a teacher's logits all slots weigh
    alike: with K = 1 the loss is cross entropy with the label
    ``index[..., 0]``.

    reduction: "none" gives float32 [...], "sum" their sum, "mean" the sum
    divided by the number of rows that have a slot (at least 1).  T^2 keeps
    gradients of one size over temperatures.  Differentiable in logits alone;
    K at most 1024.  On the CPU, and while a call is traced or transformed,
    the formula is run by torch.  Runs on the current stream of the logits'
    device; can be captured into a graph.  Results do not depend on the run.
    """
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction {reduction!r}: one of {', '.join(REDUCTIONS)}")
    if not 1e-4 <= temperature <= 1e4:
        raise ValueError(f"temperature {temperature}: wanted 1e-4 to 1e4")
    if logits.dim() < 1 or logits.shape[-1] == 0:
        raise ValueError(f"logits {tuple(logits.shape)} have no classes")
    if index.dim() < 1 or index.shape[:-1] != logits.shape[:-1]:
        raise ValueError(f"index {tuple(index.shape)} does not fit logits {tuple(logits.shape)}")
    if teacher is not None and teacher.shape != index.shape:
        raise ValueError(f"teacher {tuple(teacher.shape)} does not fit index {tuple(index.shape)}")
    if index.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"index is {index.dtype}: wanted int32 or int64")
    if not logits.is_floating_point():
        raise TypeError(f"logits are {logits.dtype}: wanted floats")
    if teacher is not None and not teacher.is_floating_point():
        raise TypeError(f"teacher is {teacher.dtype}: wanted floats")
    if teacher is not None and teacher.requires_grad:
        raise ValueError("the teacher has no gradient here: detach its logits")
    top = index.shape[-1]
    if top > MOST_SLOTS:
        raise ValueError(f"{top} slots: at most {MOST_SLOTS}")
    _native.same_device(logits=logits, index=index, teacher=teacher)
    if not _native.on_gpu(logits, index, teacher) or logits.numel() == 0 or top == 0:
        return _plain(logits, index, teacher, temperature, reduction)
    for t in (logits, teacher):
        if t is not None and t.dtype not in DTYPES:
            raise TypeError(
                f"distill_loss on a GPU takes float32, bfloat16 or float16, not {t.dtype}")
    if logits.shape[-1] >= 1 << 31:
        raise ValueError(f"{logits.shape[-1]} classes: at most 2^31 - 1")
    if _native.needs_grad(logits):
        return _Distill.apply(logits, index, teacher, temperature, reduction)
    return _forward(logits, index, teacher, temperature, REDUCTIONS[reduction], False)[0]


def _plain(logits, index, teacher, temperature, reduction):
    kind = logits.dtype if logits.dtype == torch.float64 else torch.float32
    if teacher is None:
        teacher = torch.zeros_like(index, dtype=torch.float32)
    here = (index >= 0) & (teacher != -torch.inf)
    bad = (index >= logits.shape[-1]).any(-1)
    some = here.any(-1) | bad
    t = torch.where(here, teacher.to(kind) / temperature, -torch.inf)
    t = torch.where(here.any(-1, keepdim=True), t, 0.0)
    log_p = torch.log_softmax(t, -1)
    x = torch.where(some.unsqueeze(-1), logits.to(kind) / temperature, 0.0)
    log_q = torch.log_softmax(x, -1).gather(-1, index.long().clamp(0, logits.shape[-1] - 1))
    p = torch.where(here, log_p.exp(), 0.0)
    rows = torch.where(p != 0, p * (log_p - log_q), 0.0).sum(-1) * temperature ** 2
    rows = torch.where(some, rows, 0.0) * torch.where(bad, torch.nan, 1.0)
    if reduction == "none":
        return rows
    total = rows.sum()
    return total if reduction == "sum" else total / some.sum().clamp_min(1)


def _inputs(logits, index, teacher):
    top = index.shape[-1]
    return (rows_of(logits, logits.shape[-1]), rows_of(index, top),
            None if teacher is None else rows_of(teacher, top))


def _forward(logits, index, teacher, temperature, reduction, keep):
    """The loss, and what backward needs: one buffer of the rows' log sums,
    the slots' masses and classes and the number of rows with a target."""
    x, i, t = _inputs(logits, index, teacher)
    rows, v = x.shape
    top = i.shape[1]
    device = logits.device
    chunks = _native.library().vgpu_ops_distill_chunks(rows, v, 0)
    part = (torch.empty(rows * chunks * 2, dtype=torch.float32, device=device)
            if chunks > 1 else None)
    rows_loss = torch.empty(logits.shape[:-1], dtype=torch.float32, device=device)
    loss = rows_loss
    saved = at = None
    if keep or reduction:
        saved = torch.empty(rows + 2 * rows * top + 1, dtype=torch.float32, device=device)
        at = saved.data_ptr()
    if reduction:
        loss = torch.empty((), dtype=torch.float32, device=device)
    launch("distill", _arguments(
        x, i, t, at, rows, v, top, temperature, reduction, chunks, rows_loss=rows_loss.data_ptr(),
        loss=loss.data_ptr(), part=ptr(part)), device)
    return loss, saved


def _arguments(x, i, t, at, rows, v, top, temperature, reduction, chunks, **more):
    a = DistillArgs(x=x.data_ptr(), index=ptr(i), teacher=ptr(t), ldx=x.stride(0), rows=rows, v=v,
                    dtype=DTYPES[x.dtype], top=top, chunks=chunks, reduction=reduction,
                    temperature=temperature, index_bytes=8, **more)
    if at:
        a.lse, a.slot_p = at, at + 4 * rows
        a.slot_i, a.count = at + 4 * rows * (1 + top), at + 4 * rows * (1 + 2 * top)
    if i is not None:
        a.ldi, a.index_bytes = i.stride(0), i.element_size()
    if t is not None:
        a.ldt, a.ttype = t.stride(0), DTYPES[t.dtype]
    return a


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, index, teacher, temperature, reduction):
        loss, saved = _forward(logits, index, teacher, temperature, REDUCTIONS[reduction], True)
        ctx.temperature, ctx.reduction = temperature, reduction
        ctx.save_for_backward(logits, index, teacher, saved)
        return loss

    @staticmethod
    def backward(ctx, grad):
        logits, index, teacher, saved = ctx.saved_tensors
        if torch.is_grad_enabled():
            found = _native.gradients_of(
                lambda x: _plain(x, index, teacher, ctx.temperature, ctx.reduction), (logits,),
                (True,), grad)
            return (*found, None, None, None, None)
        x = rows_of(logits, logits.shape[-1])
        rows, v = x.shape
        grad = grad.contiguous()
        dx = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        chunks = _native.library().vgpu_ops_distill_chunks(rows, v, 1)
        launch("distill", _arguments(
            x, None, None, saved.data_ptr(), rows, v, index.shape[-1], ctx.temperature,
            REDUCTIONS[ctx.reduction], chunks, dx=dx.data_ptr(), lddx=v, grad=grad.data_ptr()),
            logits.device)
        return dx, None, None, None, None
