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
