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


def tied(kind, device, dtype=torch.float32):
    """Calls whose inputs depend on each other, as (f of the operator and its
    leaves, the leaves)."""
    gen = seeded(4)
    e = normal(gen, 7, 5, device=device).to(dtype).requires_grad_()
    b = normal(gen, 7, device=device).to(dtype).requires_grad_()
    if kind == "same":
        return lambda op: op(e, e, b), [e, b]
    if kind == "embedding":
        return lambda op: op(torch.tanh(e[:3]), e, b), [e, b]
    if kind == "bias":
        return lambda op: op(e[:4], e, e.sum(1) * b), [e, b]

    def norm(op):
        w = e[0] * 2
        return op(torch.sin(e[:3] * w), w, e[1])
    return norm, [e]


def derivatives(call, op, leaves):
    """First gradients with a graph, and the second ones of their squares."""
    y = call(op)
    up = torch.linspace(-1, 2, y.numel(), device=y.device, dtype=y.dtype).view(y.shape)
    first = torch.autograd.grad(y, leaves, up, create_graph=True)
    return [*(g.detach() for g in first),
            *torch.autograd.grad(sum((g * g).sum() for g in first), leaves, materialize_grads=True)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["same", "embedding", "bias", "norm"])
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_gradients_with_a_graph_where_inputs_depend_on_each_other(kind, act):
    f = {"none": lambda z: z, "gelu": F.gelu}[act]
    if kind == "norm":
        ours = lambda *t: ops.layer_norm(*t)  # noqa: E731
        plain = lambda x, w, b: F.layer_norm(x, (5,), w, b)  # noqa: E731
    else:
        ours = lambda *t: ops.linear(*t, activation=act)  # noqa: E731
        plain = lambda *t: f(F.linear(*t))  # noqa: E731
    call, leaves = tied(kind, "cuda")
    got = derivatives(call, ours, leaves)
    call, leaves = tied(kind, "cpu", torch.float64)
    for a, b in zip(got, derivatives(call, plain, leaves)):
        # sums of fewer than 2000 products of ordinary size, twice differentiated
        assert (a.double().cpu() - b).norm() <= 2000 * U * b.norm()


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_gradients_of_stop_at_each_input(device):
    from k8s_device_plugin_amd.ops import _native

    leaf = normal(seeded(), 6, 5, device=device).requires_grad_()
    x = torch.tanh(leaf[:3])
    for inputs in ((x, leaf), (leaf, leaf)):
        grad = torch.ones(inputs[0].shape[0], 6, device=device)
        got = _native.gradients_of(F.linear, inputs, (True, True), grad)
        apart = [t.detach().requires_grad_() for t in inputs]
        for a, b in zip(got, torch.autograd.grad(F.linear(*apart), apart, grad)):
            assert torch.equal(a, b) and a.requires_grad
        none, w = _native.gradients_of(F.linear, inputs, (False, True), grad)
        assert none is None and torch.equal(w, got[1])


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_calls_under_a_dispatch_mode_run_the_formula(device):
    """What records or counts torch's operations sees the whole call."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode

    gen = seeded()
    x, w = normal(gen, 6, 8, device=device), normal(gen, 5, 8, device=device)
    index = torch.zeros(6, 1, dtype=torch.long, device=device)

    def f(x, w):
        y = ops.linear(x, w, activation="gelu")
        return y, ops.layer_norm(x), ops.distill_loss(y, index)

    def gradients(x, w):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        y, h, loss = f(x, w)
        return torch.autograd.grad((y.sum(), (h * h * h).sum(), loss), (x, w))

    a, b = normal(gen, 6, 8, device=device), normal(gen, 5, 8, device=device)
    for g in (f, gradients):
        traced = make_fx(g)(x, w)
        for got, want in zip(traced(a, b), g(a, b)):
            assert (got - want).abs().max() <= 256 * U * (1 + want.abs().max())
    with FlopCounterMode(display=False) as counter:
        ops.linear(x, w)
    assert counter.get_total_flops() == 2 * 6 * 8 * 5
    # a backward pass alone, whose graph was made outside: the formula is run again
    leaf = x.clone().requires_grad_()
    y = ops.linear(leaf, w)
    with FlopCounterMode(display=False) as counter:
        got, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert counter.get_total_flops() >= 2 * 6 * 8 * 5 and not got.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", ["eager", "another graph"])
@pytest.mark.parametrize("rows,v", [(20, 1000), (600, 9001)])
def test_distill_backward_captured_without_its_forward(dtype, how, rows, v):
    """A captured backward pass writes its gradient on every replay, whatever
    the upstream gradient was before and whatever was done to the last one."""
    logits, index, teacher = distill_inputs(rows, v, 3, dtype, "cuda")
    leaf = logits.requires_grad_()
    up = torch.ones((), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    first, graph = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()

    def loss_of():
        return ops.distill_loss(leaf, index, teacher, temperature=2.0)

    with torch.cuda.stream(side):
        want, = torch.autograd.grad(loss_of(), leaf)
        twice, = torch.autograd.grad(loss_of(), leaf, 2 * up)
        torch.cuda.synchronize()
        if how == "eager":
            loss = loss_of()
        else:
            with torch.cuda.graph(first, stream=side):
                loss = loss_of()
            first.replay()
        with torch.cuda.graph(graph, stream=side):
            grad, = torch.autograd.grad(loss, leaf, up, retain_graph=True)
        for scale, expected in ((1, want), (2, twice), (1, want), (1, want), (2, twice)):
            up.fill_(scale)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(grad, expected)
            grad.mul_(7)  # the caller's, as a clipped gradient is
            torch.randn(1 << 20, device="cuda").sum()
    torch.cuda.current_stream().wait_stream(side)


MANY = (1 << 21) + 1  # rows of fp32: one more than 8 MiB of them


def linear_work(m, n, k, dtype=0, **how):
    import ctypes

    from k8s_device_plugin_amd.ops import _native

    a = dict(x=4096, w=4096, dy=4096, dx=4096, dw=4096, db=4096, m=m, n=n, k=k, xs0=k, xs1=1, ws0=k,
             ws1=1, lddy=n, dtype=dtype)
    return _native.library().vgpu_ops_linear_work(ctypes.byref(_native.LinearArgs(**{**a, **how})))


@pytest.mark.parametrize("dtype,m", [(0, MANY), (1, 2 * MANY), (2, 2 * MANY)])
@pytest.mark.parametrize("n,k", [(1, 64), (2, 64), (16, 64), (17, 64), (257, 64), (300, 64), (1030, 64),
                                 (64, 1), (64, 5), (1, 1), (33, 2)])
def test_linear_backward_of_many_rows_has_a_plan(dtype, m, n, k):
    assert linear_work(m, n, k, dtype) >= 0
    assert linear_work(m, n, k, dtype, xs0=1, xs1=m) >= 0       # tokens contiguous
    assert linear_work(m, n, k, dtype, xs0=1, xs1=m + 3) >= 0
    assert linear_work(m, n, k, dtype, xs0=0) >= 0              # one row for all


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,m", [(torch.float32, MANY), (torch.bfloat16, 2 * MANY)])
@pytest.mark.parametrize("n,k,columns", [(1, 64, False), (16, 64, False), (257, 64, False),
                                         (64, 64, True), (64, 1, False), (40, 3, True)])
def test_linear_backward_of_many_rows(dtype, m, n, k, columns):
    """Small whole numbers: their sums are exact in any order."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    whole = lambda *s: torch.randint(-1, 2, s, generator=gen, device="cuda", dtype=torch.int8).to(dtype)  # noqa: E731
    x = whole(k, m).t() if columns else whole(m, k)
    x.requires_grad_()
    w, b = whole(n, k).requires_grad_(), whole(n).requires_grad_()
    y = ops.linear(x, w, b)
    g = whole(m, n)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
    sums, column = torch.zeros(n, k, dtype=torch.float64, device="cuda"), 0
    for part in range(0, m, 1 << 18):
        at = slice(part, min(m, part + (1 << 18)))
        sums += g[at].double().t() @ x.detach()[at].double()
        column = column + g[at].double().sum(0)
    assert torch.equal(dw, sums.to(dtype)) and torch.equal(db, column.to(dtype))
    for at in (slice(0, 70), slice(m // 2, m // 2 + 70), slice(m - 70, m)):
        assert torch.equal(dx[at], (g[at].double() @ w.detach().double()).to(dtype))
        assert torch.equal(y.detach()[at], (x.detach()[at].double() @ w.detach().double().t()
                                            + b.detach().double()).to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 3])
def test_linear_outputs_past_one_axis_of_a_launch(m):
    """16-bit weights whose rows start on 2 bytes, and more strips of outputs
    than a launch for few rows holds."""
    n = (1 << 27) + 21
    w = torch.randint(-8, 9, (n, 1), device="cuda", dtype=torch.int8).to(torch.float16)
    x = torch.arange(1, m + 1, device="cuda", dtype=torch.float16)[:, None]
    y = ops.linear(x, w)
    assert torch.equal(y, x * w.t())


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_linear_inputs_that_no_gradient_takes_may_be_changed(device, act):
    gen = seeded()
    x, w, b = (normal(gen, *s, device=device) for s in ((3, 8), (5, 8), (5,)))
    g = normal(gen, 3, 5, device=device)

    def gradients(learnt, change):
        t = {"x": x.clone(), "w": w.clone(), "b": b.clone()}
        leaves = [t[n].requires_grad_() for n in learnt]
        t["x"] = t["x"] * 1
        y = ops.linear(t["x"], t["w"], t["b"], activation=act)
        with torch.no_grad():
            for n in change:
                t[n].mul_(3)
        return torch.autograd.grad(y, leaves, g)

    bent = act in ("gelu", "silu")
    for learnt, change in (("wb", "b" if bent else "wb"), ("x", "b" if bent else "xb"), ("xwb", "b"),
                           ("b", "b" if bent else "xwb")):
        for a, c in zip(gradients(learnt, change), gradients(learnt, "")):
            assert torch.equal(a, c), (learnt, change)
    if not bent:
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            gradients("xw", "w")


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_norm_bias_may_be_changed(device):
    x, b = normal(seeded(), 3, 8, device=device).requires_grad_(), torch.zeros(8, device=device)
    b.requires_grad_()
    y = ops.layer_norm(x, None, b)
    z = ops.layer_norm(x, None, b)
    with torch.no_grad():
        b.add_(1)
    for a, c in zip(torch.autograd.grad(y.sin().sum(), (x, b), create_graph=True),
                    torch.autograd.grad(z.sin().sum(), (x, b))):
        assert (a - c).abs().max() <= 400 * U


@pytest.mark.gpu
def test_linear_second_derivative_needs_the_bias_of_a_bent_slope():
    x, w = (normal(seeded(), *s, device="cuda").requires_grad_() for s in ((3, 8), (5, 8)))
    b = torch.zeros(5, device="cuda")
    y = ops.linear(x, w, b, activation="gelu")
    b.add_(1)
    torch.autograd.grad(y.sum(), x, retain_graph=True)
    with pytest.raises(RuntimeError, match="bias has been changed"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("learnt", [(0,), (1,), (2,), (0, 1), (0, 2), (1, 2), (0, 1, 2)])
def test_linear_derivatives_of_some_inputs(device, act, learnt):
    """First and second derivatives, with the other inputs frozen."""
    gen = seeded(9)
    f = {"none": lambda z: z, "relu": F.relu, "silu": F.silu}[act]
    tensors = [normal(gen, *s) for s in ((2, 3, 8), (5, 8), (5,))]
    tensors[0][0, 0] = 0  # rows whose sum is the bias alone

    def both(op, device, dtype):
        t = [a.to(device=device, dtype=dtype, copy=True) for a in tensors]
        leaves = [t[i].requires_grad_() for i in learnt]
        y = op(*t)
        up = torch.linspace(-1, 2, y.numel(), device=device, dtype=dtype).view(y.shape).requires_grad_()
        first = torch.autograd.grad(y, leaves, up, create_graph=True)
        plain = torch.autograd.grad(y, leaves, up, retain_graph=True)
        second = torch.autograd.grad(sum((g * g).sum() for g in first), [*leaves, up],
                                     materialize_grads=True)
        return [g.detach() for g in (*first, *plain, *second)]

    got = both(lambda *t: ops.linear(*t, activation=act), device, torch.float32)
    for a, b in zip(got, both(lambda *t: f(F.linear(*t)), "cpu", torch.float64)):
        assert a.shape == b.shape and (a.double().cpu() - b).norm() <= 2000 * U * b.norm()


@pytest.mark.parametrize("device,dtype", PAIRS)
@pytest.mark.parametrize("t", [0.25, 0.5, 1.0])
@pytest.mark.parametrize("top,v", [(1, 50), (3, 50), (1, 9000)])
def test_distill_named_class_at_the_students_lowest_value(device, dtype, t, top, v):
    """Where the loss is below fp32's greatest it is that, though x / T is not."""
    logits, index, teacher = distill_inputs(3, v, top, dtype, device, seed=v)
    low = torch.finfo(dtype).min
    logits[1, index[1]] = low
    logits[2, index[2, 0]] = low
    leaf = logits.clone().requires_grad_()
    loss = ops.distill_loss(leaf, index, teacher, temperature=t, reduction="none")
    s = logits.double() / t
    q = torch.log_softmax(s, 1).gather(1, index)
    p = torch.softmax(teacher.double() / t, 1)
    want = t * t * (p * (p.log() - q)).sum(1)
    # masses off by p_off of themselves, products and sums by a few u
    far = (teacher.double() / t).abs().amax(1)
    off = U * (8 * far + 64 + v / 128 + top) * (t * t * (p * (p.log().abs() + q.abs())).sum(1) + 1)
    within(loss.detach(), want, off)
    grad, = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
    exact, slack = distill_gradient(logits.masked_fill(logits == low, -INF), index, teacher, t, 1.0)
    # 16-bit logits: the hardware's power of two gives 0 for a result below 2^-126
    within(grad[1:], exact[1:], slack[1:] + (0 if dtype == torch.float32 else t * 2.0 ** -126))


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_calls_under_a_function_mode_run_the_formula(device):
    from torch.overrides import TorchFunctionMode

    class Names(TorchFunctionMode):
        def __torch_function__(self, f, types, args=(), kwargs=None):
            seen.append(getattr(f, "__name__", str(f)))
            return f(*args, **(kwargs or {}))

    gen, seen = seeded(), []
    x, w = normal(gen, 6, 700, device=device), normal(gen, 5, 700, device=device)
    index = torch.zeros(6, 1, dtype=torch.long, device=device)
    for call, name in ((lambda: ops.linear(x, w), "linear"), (lambda: ops.layer_norm(x), "layer_norm"),
                       (lambda: ops.distill_loss(x, index), "gather")):
        with Names():
            call()
        assert name in seen
        want = call()
        with torch.device(device):  # a default device is a mode too, which looks on at nothing
            assert torch.equal(call(), want)


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_linear_with_a_gradient_in_the_residual_alone(device, act):
    gen = seeded()
    x, w = normal(gen, 3, 8, device=device), normal(gen, 5, 8, device=device)
    r = normal(gen, 3, 5, device=device).requires_grad_()
    y = ops.linear(x, w, activation=act, residual=r)
    up = normal(gen, 3, 5, device=device).requires_grad_()
    for graph in (False, True):
        got, = torch.autograd.grad(y, r, up, retain_graph=True, create_graph=graph)
        assert torch.equal(got, up)


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_backward_alone_under_a_dispatch_mode(device):
    from torch.utils.flop_counter import FlopCounterMode

    gen = seeded()
    x, w, b = (normal(gen, *s, device=device).requires_grad_() for s in ((6, 12), (12,), (12,)))
    index = torch.arange(6, device=device)[:, None]
    for y in (ops.layer_norm(x, w, b, groups=3), ops.layer_norm(x, None, b), ops.layer_norm(x),
              ops.distill_loss(x, index), ops.distill_loss(x, index, reduction="none", temperature=2.0)):
        leaves = [t for t in (x, w, b) if t is x or (y.dim() == 2 and torch.autograd.grad(
            y.sum(), t, retain_graph=True, allow_unused=True)[0] is not None)]
        up = normal(gen, *(y.shape or (1,)), device=device).reshape(y.shape)
        want = torch.autograd.grad(y, leaves, up, retain_graph=True)
        with FlopCounterMode(display=False):
            got = torch.autograd.grad(y, leaves, up)
        for a, c in zip(got, want):
            # two evaluations of sums of fewer than 32 terms of ordinary size
            assert a.dtype == c.dtype and not a.requires_grad and (a - c).abs().max() <= 400 * U
