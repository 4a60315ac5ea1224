"""The head operators where a value, a size or a way of calling is at an edge.

Bounds are counted as in test_head_ops.py: u = 2^-24 for each fp32 operation,
half a step of the tensor's type for each value that is stored.
"""
import pytest
import torch
import torch.nn.functional as F

from k8s_device_plugin_amd import ops
from test_head_ops import (DTYPES, GPU, PAIRS, U, check_distill, distill_inputs, native,  # noqa: F401
                           normal, seeded, within)

INF = float("inf")


def distill_gradient(logits, index, teacher, t, each):
    """In 64 bits, from q - p: finite wherever a softmax is.  `each` is the
    loss's weight of a row; second, the bound of what fp32 may be off by."""
    s = logits.detach().double() / t
    lse = torch.logsumexp(s, 1, keepdim=True)
    q = (s - lse).exp()
    p = torch.softmax(teacher.double() / t, 1)
    want = (q.scatter_add(1, index.long(), -p)) * (each * t)
    finite = s.nan_to_num(0, 0, 0)
    most = finite.abs().amax(1, keepdim=True)
    far = (teacher.double() / t).abs().amax(1, keepdim=True)
    lse_off = U * (8 * most + 32 + s.shape[1] / 128)
    p_off = U * (8 * far + 32 + index.shape[1])
    mass = q + want.abs() / (each * t)
    return want, each * t * (q * (lse_off + 8 * U * (4 + (finite - lse).abs())) + mass * (p_off + 8 * U))


@pytest.mark.parametrize("device,dtype", PAIRS)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("top,v,t", [(1, 50, 1.0), (3, 50, 2.0), (1, 9000, 1.0), (70, 515, 0.5)])
def test_distill_all_named_classes_masked_in_the_student(device, dtype, reduction, top, v, t):
    """Every class that a row names has a logit of -inf: the loss is +inf, not
    NaN, and the gradient stays the softmax less the teacher's masses."""
    logits, index, teacher = distill_inputs(4, v, top, dtype, device, seed=v)
    logits[1, index[1]] = -INF
    clean = ops.distill_loss(logits[[0, 2, 3]], index[[0, 2, 3]], teacher[[0, 2, 3]], temperature=t,
                             reduction="none")
    leaf = logits.clone().requires_grad_()
    loss = ops.distill_loss(leaf, index, teacher, temperature=t, reduction=reduction)
    if reduction == "none":
        assert torch.equal(loss.detach()[[0, 2, 3]], clean)
    assert (loss if reduction != "none" else loss[1]) == INF
    if top == 1:
        want = F.cross_entropy(logits.double(), index[:, 0], reduction=reduction)
        assert torch.equal(want.isinf(), loss.detach().isinf().reshape(want.shape))
    each = 0.25 if reduction == "mean" else 1.0
    grad, = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
    within(grad, *distill_gradient(logits, index, teacher, t, each))
    half, = torch.autograd.grad(
        ops.distill_loss(leaf, index, teacher, temperature=t, reduction=reduction), leaf,
        torch.full_like(loss, 0.5))
    within(half, *distill_gradient(logits, index, teacher, t, each / 2))


@pytest.mark.parametrize("device,dtype", PAIRS)
@pytest.mark.parametrize("act", ["gelu", "silu", "relu"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("m,n", [(3, 24), (40, 520), (300, 520)])
def test_linear_value_before_the_activation_past_the_types_range(device, dtype, act, residual, m, n):
    """Sums of +-1.4e6, which fp16 cannot hold: the slope is 1 or 0 there, as
    it is in fp32, and the gradients are finite."""
    k = 16
    sign = torch.ones(n)
    sign[1::2] = -1
    x = torch.full((m, k), 300.0, device=device, dtype=dtype).requires_grad_()
    w = (300 * sign)[:, None].expand(n, k).to(device=device, dtype=dtype).contiguous().requires_grad_()
    b = torch.zeros(n, device=device, dtype=dtype, requires_grad=True)
    r = torch.zeros(m, n, device=device, dtype=dtype) if residual else None
    y = ops.linear(x, w, b, activation=act, residual=r)
    assert (y[:, ::2] == torch.full((), 300.0 * 300 * k, dtype=torch.float64).to(dtype).to(device)).all()
    assert (y[:, 1::2] == 0).all()
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.full_like(y, 0.125))
    # sums of multiples of 1/8 below 2^21: exact, and stored with one rounding
    on = (sign > 0).double().to(device)
    assert torch.equal(dx, (0.125 * 300 * on.sum()).expand(m, k).to(dtype))
    assert torch.equal(dw, (0.125 * 300 * m * on)[:, None].expand(n, k).to(dtype))
    assert torch.equal(db, (0.125 * m * on).to(dtype))


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.gpu
def test_linear_value_before_the_activation_past_bfloat16s_range(act):
    """2^126 x 3.97 and a bias: finite in fp32, rounded past bf16's greatest."""
    big = 1.9921875 * 2.0 ** 63
    x = torch.full((5, 1), big, device="cuda", dtype=torch.bfloat16)
    w = torch.tensor([[big], [-big]] * 12, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    b = torch.tensor([2.3e36, -2.3e36] * 12, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = ops.linear(x, w, b, activation=act)
    assert (y[:, ::2] == INF).all() and (y[:, 1::2] == 0).all()
    dw, db = torch.autograd.grad(y, (w, b), torch.ones_like(y))
    on = torch.tensor([1.0, 0.0] * 12, device="cuda", dtype=torch.float64)
    assert torch.equal(dw[:, 0], (5 * big * on).bfloat16()) and torch.equal(db, (5 * on).bfloat16())


@pytest.mark.parametrize("device,dtype", PAIRS)
@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("t", [0.25, 0.5, 1.0, 3.0])
def test_distill_teacher_at_the_lowest_value(device, dtype, reduction, t):
    """Slots at the type's lowest value have no mass beside an ordinary one,
    and weigh alike where there is no other: dividing by T empties no row."""
    logits, index, teacher = distill_inputs(6, 60, 5, dtype, device)
    same = teacher.clone()
    low = torch.finfo(dtype).min
    teacher[1], same[1] = low, 0.0
    teacher[2, :2], teacher[2, 2:] = low, -INF
    same[2, :2], same[2, 2:] = 0.0, -INF
    teacher[3, 1:], same[3, 1:] = low, -INF
    teacher[4], same[4] = -low, 0.0
    teacher[5, 0] = -INF
    same[5, 0] = -INF

    def both(teacher):
        leaf = logits.clone().requires_grad_()
        loss = ops.distill_loss(leaf, index, teacher, temperature=t, reduction=reduction)
        return loss.detach(), torch.autograd.grad(loss, leaf, torch.ones_like(loss))[0]

    check_distill(logits, index, same, t, reduction)
    for a, b in zip(both(teacher), both(same)):
        assert torch.equal(a, b)
