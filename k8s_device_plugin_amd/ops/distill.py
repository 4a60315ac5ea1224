"""Distillation from a teacher's top logits; with one slot, cross entropy.

    p = softmax(teacher / T) over a row's slots
    q = softmax(logits / T) over the vocabulary
    loss = T^2 sum_k p_k (log p_k - log q[index_k])

The kernels are csrc/ops/distill.hip; the softmax's maximum and sum are held
in fp32.
"""
from __future__ import annotations

import math

import torch

from . import _native
from ._native import DTYPES, DistillArgs, launch, ptr, rows_of

REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
MOST_SLOTS = 1024


def distill_loss(logits, index, teacher=None, *, temperature=1.0, reduction="mean",
                 scale=1.0):
    """The loss of ``logits`` [..., V] against a teacher whose top classes
    are ``index`` [..., K] (int32 or int64) with logits ``teacher`` [..., K].

    A slot with a negative index, or a teacher's logit of -inf, is empty; a
    row whose slots are all empty has loss 0 and gradient 0.  A class that is
    named twice counts with both masses.  An index of V or more makes the
    row's loss and gradient NaN.  Without a teacher's logits all slots weigh
    alike: with K = 1 the loss is cross entropy with the label
    ``index[..., 0]``.

    reduction: "none" gives float32 [...], "sum" their sum, "mean" the sum
    divided by the number of rows that have a slot (at least 1), times
    ``scale``.  T^2 keeps gradients of one size over temperatures.
    Differentiable in logits alone; K at most 1024.

    Where a gradient is wanted of a loss that is one number, it is written
    along with the loss, for an upstream gradient of 1, and held until
    backward (not where only one of the two passes is captured into a graph, or
    each into its own).  Another upstream gradient costs a second writing: a factor that
    is known before, as 1/n for n accumulated steps, belongs in ``scale``.

    On the CPU, and while a call is traced or transformed, the formula is run
    by torch.  Runs on the current stream of the logits' device; can be
    captured into a graph.  Results do not depend on the run.
    """
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction {reduction!r}: one of {', '.join(REDUCTIONS)}")
    if not math.isfinite(scale) or (scale != 1 and reduction == "none"):
        raise ValueError(f"scale {scale} with reduction {reduction!r}")
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
    _native.same_device("logits index teacher", logits, index, teacher)
    if not _native.on_gpu(logits, index, teacher) or logits.numel() == 0 or top == 0:
        return _plain(logits, index, teacher, temperature, reduction, scale)
    for t in (logits, teacher):
        if t is not None and t.dtype not in DTYPES:
            raise TypeError(
                f"distill_loss on a GPU takes float32, bfloat16 or float16, not {t.dtype}")
    if logits.shape[-1] >= 1 << 31:
        raise ValueError(f"{logits.shape[-1]} classes: at most 2^31 - 1")
    if _native.needs_grad(logits):
        return _Distill.apply(logits, index, teacher, temperature, reduction, scale)
    return _forward(logits, index, teacher, temperature, REDUCTIONS[reduction], scale, False)[0]


def _plain(logits, index, teacher, temperature, reduction, scale):
    kind = logits.dtype if logits.dtype == torch.float64 else torch.float32
    if teacher is None:
        teacher = torch.zeros_like(index, dtype=torch.float32)
    here = (index >= 0) & (teacher != -torch.inf)
    bad = (index >= logits.shape[-1]).any(-1)
    some = here.any(-1) | bad
    t = teacher.to(torch.promote_types(teacher.dtype, kind)).masked_fill(~here, -torch.inf)
    t = torch.where(here.any(-1, keepdim=True), t, 0.0)
    if index.shape[-1]:  # so that no finite logit leaves its range
        t = (t - t.amax(-1, keepdim=True)) / temperature
    log_p = torch.log_softmax(t, -1).to(kind)
    x = torch.where(some.unsqueeze(-1), logits.to(kind), 0.0)
    most = x.detach().amax(-1, keepdim=True)  # so that no finite logit leaves its range
    x = x - torch.where(most.isfinite(), most, 0.0)
    lse = torch.logsumexp(x / temperature, -1, keepdim=True)
    t_log_q = x.gather(-1, index.long().clamp(0, logits.shape[-1] - 1)) - temperature * lse
    tp = torch.where(here, log_p.exp(), 0.0) * temperature
    rows = torch.where(tp != 0, tp * (temperature * log_p - t_log_q), 0.0).sum(-1)
    rows = torch.where(some, rows, 0.0) * torch.where(bad, torch.nan, 1.0)
    if reduction == "none":
        return rows
    total = rows.sum() * scale
    return total if reduction == "sum" else total / some.sum().clamp_min(1)


def _inputs(logits, index, teacher):
    top = index.shape[-1]
    return (rows_of(logits, logits.shape[-1]), rows_of(index, top),
            None if teacher is None else rows_of(teacher, top))


def _forward(logits, index, teacher, temperature, reduction, scale, keep):
    """The loss; and, to keep for backward, a buffer of the rows' states and
    log sums, the slots' masses and classes and the counts of rows with a
    target, and the gradient for an upstream gradient of 1, where writing it
    now is cheapest."""
    x, i, t = _inputs(logits, index, teacher)
    rows, v = x.shape
    top = i.shape[1]
    device = logits.device
    chunks = _native.plan("distill_chunks", rows, v, 0)
    # one workgroup a row has it in registers when its gradient can be
    # written; few long rows are better cut in pieces, and wait for backward
    dx = logits.new_empty(logits.shape) if keep and reduction and chunks == 1 else None
    loss = torch.empty(() if reduction else logits.shape[:-1], dtype=torch.float32, device=device)
    # behind what is kept: the rows' losses, where their sum is asked for, and
    # the chunks' maxima and sums
    kept = rows * (4 + 2 * top if keep else 2) + (rows + 15) // 16
    saved = torch.empty(kept + (rows if reduction else 0) + (2 * rows * chunks if chunks > 1 else 0),
                        dtype=torch.float32, device=device)
    at = saved.data_ptr() + 4 * kept
    rows_loss = at if reduction else loss.data_ptr()
    part = (at + (4 * rows if reduction else 0)) if chunks > 1 else None
    launch("distill", device, DistillArgs(
        x.data_ptr(), i.data_ptr(), ptr(t), ptr(dx), None, rows_loss,
        *_rows(saved, rows, top, keep, loss.data_ptr()), part, x.stride(0), v, i.stride(0),
        0 if t is None else t.stride(0), rows, v, DTYPES[x.dtype],
        0 if t is None else DTYPES[t.dtype], i.element_size(), top, chunks, reduction, 0,
        temperature, scale))
    return loss, saved, dx


def _rows(saved, rows, top, keep, loss):
    """Where the kernels find what is held of the rows; `state` to `slot_i`."""
    at, row = saved.data_ptr(), 4 * rows
    if not keep:
        return at, at + row, None, None, None, loss, at + 2 * row, None
    slots = at + 4 * row
    end = slots + 2 * top * row
    return at, at + row, at + 2 * row, at + 3 * row, slots, loss, end, slots + top * row


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, index, teacher, temperature, reduction, scale):
        ctx.how = temperature, reduction, scale
        loss, saved, ctx.dx = _forward(logits, index, teacher, temperature, REDUCTIONS[reduction],
                                       scale, True)
        ctx.capture = None if ctx.dx is None else _native.capture(logits.device)
        ctx.save_for_backward(logits, index, teacher, saved)
        return loss

    @staticmethod
    def backward(ctx, grad):
        logits, index, teacher, saved = ctx.saved_tensors
        # handed out once: what a caller does to it must not reach a second
        # backward pass, which writes its own
        dx, ctx.dx = ctx.dx, None
        # nor must it reach a replay of this pass alone, which has to write its
        # gradient each time
        if dx is not None and _native.capture(logits.device) != ctx.capture:
            dx = None
        if _native.formula_backward():
            found = _native.gradients_of(lambda x: _plain(x, index, teacher, *ctx.how), (logits,),
                                         (True,), grad)
            return (*found, None, None, None, None, None)
        x = rows_of(logits, logits.shape[-1])
        rows, v = x.shape
        grad = grad.resolve_neg().contiguous()
        temperature, reduction, scale = ctx.how
        top, written = index.shape[-1], dx is not None
        if not written:
            dx = logits.new_empty(logits.shape)
        launch("distill", logits.device, DistillArgs(
            x.data_ptr(), None, None, dx.data_ptr(), grad.data_ptr(), None,
            *_rows(saved, rows, top, True, None), None, x.stride(0), v, 0, 0, rows, v,
            DTYPES[x.dtype], 0, 8, top, _native.plan("distill_chunks", rows, v, 1),
            REDUCTIONS[reduction], written, temperature, scale))
        return dx, None, None, None, None, None
