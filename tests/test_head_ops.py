"""The head operators: linear, layer_norm and distill_loss.

Numbers are compared with the formula in 64 bits, element by element, against
bounds that count what the kernels round: u = 2^-24 for each fp32 operation
(a sum of n terms is off by at most n u times the sum of their sizes), half a
step of the tensor's type for each value that is stored.  On the CPU the same
entry points run the plain formula, which is held to the same bounds in fp32.
"""
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

from k8s_device_plugin_amd import ops

REPO = Path(__file__).resolve().parent.parent
U = 2.0 ** -24
CSRC = REPO / "k8s_device_plugin_amd" / "csrc"
GPU = pytest.param("cuda", marks=pytest.mark.gpu)
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def native():
    if not (CSRC / "libvgpu_ops.so").exists():
        subprocess.run(["make", "libvgpu_ops.so"], cwd=CSRC, check=True, capture_output=True)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half a step of the smallest numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def within(got, want, slack):
    """|got - want| <= slack before storing, plus the rounding of the store."""
    bound = slack + half_step(got.dtype) * (want.abs() + slack) + least(got.dtype)
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (
        f"{int(bad.sum())} of {bad.numel()} off, worst {float((off / bound).nan_to_num(9e9).max()):.3g} "
        f"bounds, first at {bad.nonzero()[0].tolist()}")


def normal(gen, *shape, dtype=torch.float32, device="cpu", scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(device=device, dtype=dtype)


def seeded(seed=0):
    return torch.Generator().manual_seed(seed)


def on(device):
    """(device, dtype) pairs: every type on the GPU, fp32 for the plain form."""
    return DTYPES if device == "cuda" else [torch.float32]


PAIRS = [("cpu", torch.float32)] + [
    pytest.param("cuda", d, marks=pytest.mark.gpu) for d in DTYPES]


# ---------------------------------------------------------------------------
# linear
# ---------------------------------------------------------------------------
ACT = {"none": lambda z: z, "relu": F.relu, "gelu": F.gelu, "silu": F.silu}
SLOPE_MOST = {"none": 1.0, "relu": 1.0, "gelu": 1.13, "silu": 1.1}   # max |act'|
BEND_MOST = {"none": 0.0, "relu": 0.0, "gelu": 0.8, "silu": 0.5}     # max |act''|


def check_linear(x, w, b, r, act, backward=True, seed=1):
    leaves = [t if t is None or not backward else t.detach().requires_grad_() for t in (x, w, b, r)]
    y = ops.linear(leaves[0], leaves[1], leaves[2], activation=act, residual=leaves[3])
    n, k = w.shape
    assert y.shape == x.shape[:-1] + (n,) and y.dtype == x.dtype and y.device == x.device
    lead = x.shape[:-1].numel()
    x64 = x.detach().double().reshape(lead, k)
    w64 = w.detach().double()
    z = x64 @ w64.t() if k else x64.new_zeros(x64.shape[0], n)
    size = x64.abs() @ w64.abs().t() if k else torch.zeros_like(z)
    if b is not None:
        z = z + b.detach().double()
        size = size + b.detach().double().abs()
    z_off = (k + 2) * U * size
    want = ACT[act](z)
    # the activation's own fp32 evaluation: at most 16 operations on |z|
    off = SLOPE_MOST[act] * z_off + (0 if act in ("none", "relu") else 16 * U) * z.abs()
    if r is not None:
        r64 = r.detach().double().reshape(-1, n)
        want = want + r64
        off = off + U * (want.abs() + r64.abs())
    within(y.detach().reshape(-1, n), want, off)
    if not backward:
        return
    g = normal(seeded(seed), *y.shape, dtype=x.dtype, device=x.device)
    used = [t for t in leaves if t is not None]
    grads = dict(zip([i for i, t in enumerate(leaves) if t is not None],
                     torch.autograd.grad(y, used, g)))
    g64 = g.double().reshape(-1, n)
    zz = z.clone().requires_grad_()
    slope = torch.autograd.grad(ACT[act](zz).sum(), zz)[0] if act != "none" else torch.ones_like(z)
    dz = g64 * slope
    # the slope at a z that was stored in the type, 24 operations of its own,
    # and dz stored in the type
    step = half_step(x.dtype)
    dz_off = torch.zeros_like(dz)
    if act != "none":
        dz_off = g64.abs() * (BEND_MOST[act] * (z_off + step * z.abs() + least(x.dtype))
                              + 24 * U * (1 + z.abs()))
        dz_off = dz_off + step * dz.abs() + least(x.dtype)
    if act == "relu":  # which side of 0 a z within its own error falls on is open
        dz_off = dz_off + g64.abs() * (z.abs() <= z_off)
    rows = max(1, dz.shape[0])
    dz_most = dz.abs() + dz_off
    within(grads[0].reshape(lead, k), dz @ w64, dz_off @ w64.abs() + (n + 2) * U * (dz_most @ w64.abs()))
    within(grads[1], dz.t() @ x64,
           dz_off.t() @ x64.abs() + (rows + 2) * U * (dz_most.t() @ x64.abs()))
    if b is not None:
        within(grads[2], dz.sum(0), dz_off.sum(0) + (rows + 2) * U * dz_most.sum(0))
    if r is not None:
        assert torch.equal(grads[3], g)


SHAPES = [(1, 1, 1), (1, 8, 16), (2, 9, 3), (3, 7, 5), (5, 256, 1000), (16, 96, 48), (17, 129, 65),
          (20, 520, 130), (33, 64, 200), (64, 64, 64), (65, 72, 264), (130, 200, 70), (257, 512, 300),
          (1, 2048, 4096), (700, 40, 700)]


@pytest.mark.parametrize("device,dtype", PAIRS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("act,bias,residual", [
    ("none", False, False), ("none", True, True), ("relu", True, False), ("relu", False, True),
    ("gelu", True, True), ("silu", True, False)])
def test_linear(device, dtype, shape, act, bias, residual):
    m, k, n = shape
    gen = seeded(m * 31 + k * 7 + n)
    make = lambda *s, scale=1.0: normal(gen, *s, dtype=dtype, device=device, scale=scale)  # noqa: E731
    check_linear(make(m, k), make(n, k, scale=k ** -0.5), make(n) if bias else None,
                 make(m, n) if residual else None, act)


@pytest.mark.parametrize("device,dtype", PAIRS)
@pytest.mark.parametrize("m", [1, 5, 40, 300])
@pytest.mark.parametrize("case", ["x_columns", "x_slice", "x_odd_start", "x_one_row", "w_columns",
                                  "w_slice", "both_columns", "r_one_row", "b_strided", "w_steps"])
def test_linear_strides(device, dtype, m, case):
    k, n = 72, 136
    gen = seeded(m)
    make = lambda *s, scale=1.0: normal(gen, *s, dtype=dtype, device=device, scale=scale)  # noqa: E731
    x, w, b, r = make(m, k), make(n, k, scale=0.1), make(n), make(m, n)
    if case in ("x_columns", "both_columns"):
        x = x.t().contiguous().t()
    if case in ("w_columns", "both_columns"):
        w = w.t().contiguous().t()
    if case == "x_slice":
        x = make(m, k + 5)[:, 3:k + 3]
    if case == "x_odd_start":
        x = make(m * k + 1)[1:].view(m, k)
    if case == "x_one_row":
        x = make(1, k).expand(m, k)
    if case == "w_slice":
        w = make(n + 3, k + 8)[2:n + 2, 8:]
    if case == "r_one_row":
        r = make(1, n).expand(m, n)
    if case == "b_strided":
        b = make(2 * n)[::2]
    if case == "w_steps":
        w = make(n, 2 * k, scale=0.1)[:, ::2]
    check_linear(x, w, b, r, "gelu")


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_linear_leading_axes_and_empty(device):
    gen = seeded()
    x = normal(gen, 2, 3, 16, device=device)
    check_linear(x, normal(gen, 8, 16, device=device), None, normal(gen, 2, 3, 8, device=device), "silu")
    check_linear(x[0, 0], normal(gen, 8, 16, device=device), normal(gen, 8, device=device), None, "none")
    check_linear(x[:0], normal(gen, 8, 16, device=device), normal(gen, 8, device=device), None, "relu")
    check_linear(x[..., :0], normal(gen, 8, 0, device=device), normal(gen, 8, device=device), None, "relu")


@pytest.mark.parametrize("device,dtype", PAIRS)
@pytest.mark.parametrize("m,k,n", [(3, 40, 24), (70, 33, 130)])
def test_linear_keeps_what_is_not_finite_in_its_row(device, dtype, m, k, n):
    gen = seeded()
    x, w = normal(gen, m, k, dtype=dtype, device=device), normal(gen, n, k, dtype=dtype, device=device)
    clean = ops.linear(x, w)
    x[1, 5], x[2, k - 1] = float("inf"), float("nan")
    y = ops.linear(x, w)
    others = [i for i in range(m) if i not in (1, 2)]
    assert torch.equal(y[others], clean[others])
    assert not y[1].isfinite().any() and y[2].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_long_sums_and_many_tiles(dtype):
    """Sizes that reach every tile, the split over k and its join."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    for m, k, n in ((2, 25088, 256), (48, 8200, 520), (96, 6000, 96), (300, 4096, 260),
                    (1030, 520, 2056), (4100, 72, 4104), (4099, 2048, 4096), (519, 3000, 8200)):
        x = torch.randn(m, k, generator=gen, device="cuda").to(dtype)
        w = (torch.randn(n, k, generator=gen, device="cuda") * k ** -0.5).to(dtype)
        b = torch.randn(n, generator=gen, device="cuda").to(dtype)
        check_linear(x, w, b, None, "gelu")


@pytest.mark.gpu
def test_linear_offsets_past_32_bits():
    """An output of 4.6 GB and a weight read past 4 GB."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(70000, 16, generator=gen, device="cuda").half()
    w = torch.randn(32832, 16, generator=gen, device="cuda").half()
    y = ops.linear(x, w)
    for rows in (slice(0, 3), slice(65530, 65540), slice(69990, 70000)):
        want = x[rows].double() @ w.double().t()
        within(y[rows], want, 18 * U * (x[rows].double().abs() @ w.double().abs().t()))
    del y
    w = torch.randn(270000, 8192, generator=gen, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(2, 8192, generator=gen, device="cuda", dtype=torch.bfloat16)
    y = ops.linear(x, w)
    far = w[-64:].double()
    within(y[:, -64:], x.double() @ far.t(), 8194 * U * (x.double().abs() @ far.t().abs()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 7, 16, 40, 300, 2100])
@pytest.mark.parametrize("pad", [1, 2, 3, 8])
@pytest.mark.gpu
def test_linear_reads_nothing_behind_its_rows(dtype, m, pad):
    """NaN lies behind every row and behind the last one, along either axis."""
    gen, device, h = seeded(m), "cuda", half_step(dtype)
    n = 44

    def inside(rows, cols, more=0):
        whole = torch.full((rows + more, cols + pad), float("nan"), device=device, dtype=dtype)
        whole[:rows, :cols] = normal(gen, rows, cols, dtype=dtype, device=device)
        return whole[:rows, :cols]

    for k in (1, 31, 130, 1277):
        x, dy = inside(m, k), inside(m, n)
        for w in (inside(n, k), inside(k, n, more=3).t()):
            leaf = [t.detach().requires_grad_() for t in (x, w)]
            y = ops.linear(*leaf)
            same = [t.detach().contiguous().requires_grad_() for t in (x, w)]
            z = ops.linear(*same)
            got = [y, *torch.autograd.grad(y, leaf, dy)]
            want = [z, *torch.autograd.grad(z, same, dy.contiguous())]
            for g, t, terms, (a, b) in zip(got, want, (k, n, m), ((x, w.t()), (dy, w), (dy.t(), x))):
                # two results e (1 + h) + s, where s is a sum's error in 32 bits:
                # they differ by 2 s + 2 h |e|, and |e| <= (|t| + s) / (1 - h)
                s = (terms + 2) * U * (a.abs().float() @ b.abs().float()).double()
                within(g.double(), t.double(), 2 * least(dtype) + 2 * s
                       + 2 * h * (t.double().abs() + s) / (1 - h))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, n, k", [(4096, 4096, 517), (4099, 1030, 3001), (513, 4096, 67)])
def test_linear_large_tiles_read_nothing_behind_their_rows(dtype, m, n, k):
    gen = seeded(k)

    def inside(rows, cols):
        whole = torch.full((rows + 1, cols + 3), float("nan"), device="cuda", dtype=dtype)
        whole[:rows, :cols] = normal(gen, rows, cols, dtype=dtype, device="cuda")
        return whole[:rows, :cols]

    x = inside(m, k)
    for w in (inside(n, k), inside(k, n).t()):
        y = ops.linear(x, w)
        # columns of 64 bits at a few places, all rows; and no NaN anywhere
        assert y.isfinite().all()
        at = torch.tensor([0, 1, 127, 128, n // 2, n - 2, n - 1], device="cuda")
        want = x.double() @ w[at].double().t().contiguous()
        s = (k + 2) * U * (x.abs().double() @ w[at].abs().double().t().contiguous())
        within(y[:, at], want, s)


@pytest.mark.gpu
def test_linear_rows_past_one_axis_of_a_launch():
    rows = (1 << 29) + 3
    x = torch.randn(1 << 20, 8, device="cuda", dtype=torch.float16).repeat(513, 1)[:rows]
    w = torch.randn(8, 8, device="cuda", dtype=torch.float16)
    y = ops.linear(x, w)
    for part in (slice(0, 5), slice(1 << 28, (1 << 28) + 5), slice(rows - 40, rows)):
        within(y[part].double(), x[part].double() @ w.double().T,
               least(torch.float16) + 2 * half_step(torch.float16) * (x[part].abs().double() @ w.abs().double().T))


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("device", ["cpu", GPU])
def test_linear_relu_drops_what_is_not_finite_where_it_is_off(device, dtype, residual):
    x = -torch.ones(3, 16, device=device, dtype=dtype)  # every sum is -16 ...
    x[1] = 1                                            # ... 16 ...
    x[2] = float("nan")                                 # ... or no number, which passes
    w = torch.ones(24, 16, device=device, dtype=dtype)
    b = torch.zeros(24, device=device, dtype=dtype, requires_grad=True)
    r = torch.zeros(3, 24, device=device, dtype=dtype) if residual else None
    dy = torch.ones(3, 24, device=device, dtype=dtype)
    dy[0, 3], dy[0, 4], dy[1, 5] = float("inf"), float("nan"), float("inf")
    db, = torch.autograd.grad(ops.linear(x, w, b, activation="relu", residual=r), b, dy)
    want = torch.full((24,), 2.0, device=device, dtype=dtype)
    want[5] = float("inf")
    assert torch.equal(db, want)


def test_linear_gradients_by_differences():
    gen = seeded()
    x, w, b, r = (normal(gen, *s).double().requires_grad_() for s in ((3, 5), (4, 5), (4,), (3, 4)))
    for act in ("none", "gelu", "silu"):
        assert torch.autograd.gradcheck(
            lambda x, w, b, r: ops.linear(x, w, b, activation=act, residual=r), (x, w, b, r))


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_linear_refusals(device):
    x, w = torch.zeros(2, 4, device=device), torch.zeros(3, 4, device=device)
    with pytest.raises(ValueError, match="activation"):
        ops.linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="does not fit"):
        ops.linear(x, w[:, :3])
    with pytest.raises(ValueError, match="bias"):
        ops.linear(x, w, torch.zeros(4, device=device))
    with pytest.raises(ValueError, match="residual"):
        ops.linear(x, w, residual=torch.zeros(1, 3, device=device))
    with pytest.raises(TypeError, match="weight is"):
        ops.linear(x, w.half())
    if device == "cuda":
        with pytest.raises(ValueError, match="different devices"):
            ops.linear(x, w.cpu())
        with pytest.raises(TypeError, match="float32, bfloat16"):
            ops.linear(x.double(), w.double())
        with pytest.raises(ValueError, match="8 MiB"):
            ops.linear(torch.zeros(1, 1 << 21, device=device), torch.zeros(1, 1 << 21, device=device))
        with pytest.raises(ValueError, match="8 MiB"):
            ops.linear(torch.zeros(1, 4, device=device),
                       torch.zeros(1 << 21, 4, device=device, requires_grad=True))


# ---------------------------------------------------------------------------
# layer_norm
# ---------------------------------------------------------------------------
def check_norm(x, w, b, groups, eps=1e-5, backward=True):
    leaves = [t if t is None or not backward else t.detach().requires_grad_() for t in (x, w, b)]
    y = ops.layer_norm(leaves[0], leaves[1], leaves[2], groups=groups, eps=eps)
    width = x.shape[-1]
    d = width // groups
    assert y.shape == x.shape and y.dtype == x.dtype
    x64 = x.detach().double().reshape(-1, groups, d)
    ones, zeros = torch.ones(groups, d, dtype=torch.float64, device=x.device), 0.0
    w64 = ones if w is None else w.detach().double().view(groups, d)
    b64 = ones * zeros if b is None else b.detach().double().view(groups, d)
    mean = x64.mean(-1, keepdim=True)
    rstd = 1 / (x64.var(-1, correction=0, keepdim=True) + eps).sqrt()
    h = (x64 - mean) * rstd
    # a value goes through at most 32 sums in its thread and 6 + 16 across
    # them: 64 u a sum, twice (mean, then squares), and a few products
    ratio = x64.abs().mean(-1, keepdim=True) * rstd
    c = 160 * U
    h_off = c * (ratio + h.abs() * (1 + ratio))
    want = h * w64 + b64
    within(y.detach().reshape(-1, width), want.flatten(1),
           (h_off * w64.abs() + 3 * U * ((h * w64).abs() + b64.abs())).flatten(1))
    if not backward:
        return
    g = normal(seeded(3), *x.shape, dtype=x.dtype, device=x.device)
    used = [t for t in leaves if t is not None]
    grads = dict(zip([i for i, t in enumerate(leaves) if t is not None],
                     torch.autograd.grad(y, used, g)))
    g64 = g.double().reshape(-1, groups, d)
    a = g64 * w64
    ma, mah = a.mean(-1, keepdim=True), (a * h).mean(-1, keepdim=True)
    dx = rstd * (a - ma - h * mah)
    sizes = a.abs() + a.abs().mean(-1, keepdim=True) + h.abs() * (a * h).abs().mean(-1, keepdim=True)
    dx_off = rstd * (c * (1 + ratio) * sizes + h_off * mah.abs()
                     + h.abs() * (a.abs() * h_off).mean(-1, keepdim=True))
    within(grads[0].reshape(-1, width), dx.flatten(1), dx_off.flatten(1))
    rows = max(1, x64.shape[0])
    if w is not None:
        within(grads[1], (g64 * h).sum(0).flatten(),
               ((g64.abs() * h_off).sum(0) + (rows + 2) * U * (g64 * h).abs().sum(0)).flatten())
    if b is not None:
        within(grads[2], g64.sum(0).flatten(), ((rows + 2) * U * g64.abs().sum(0)).flatten())


@pytest.mark.parametrize("device,dtype", PAIRS)
@pytest.mark.parametrize("rows,groups,d", [
    (1, 1, 1), (1, 1, 8), (2, 32, 8), (3, 1, 7), (5, 4, 65), (9, 1, 512), (2, 1, 513), (7, 1, 1024),
    (130, 2, 1030), (4, 1, 2049), (3, 1, 5001), (2, 1, 8192), (2, 1, 12000), (2, 1, 16385),
    (1, 1, 32768), (2100, 1, 24), (600, 1, 2056)])
def test_norm(device, dtype, rows, groups, d):
    gen = seeded(rows + d)
    make = lambda *s: normal(gen, *s, dtype=dtype, device=device)  # noqa: E731
    width = groups * d
    check_norm(make(rows, width) * 1.5 + 0.5, make(width), make(width), groups)


@pytest.mark.parametrize("device,dtype", PAIRS)
def test_norm_forms(device, dtype):
    gen = seeded()
    make = lambda *s, to=dtype: normal(gen, *s, dtype=to, device=device)  # noqa: E731
    check_norm(make(4, 40), None, None, 1)
    check_norm(make(4, 40), make(40), None, 2)
    check_norm(make(4, 40), None, make(40), 1)
    check_norm(make(4, 41), make(41, to=torch.float32), make(41, to=torch.float32), 1)
    check_norm(make(4, 47)[:, 3:44], make(41), make(82)[::2], 1)
    check_norm(make(41, 6).t(), make(41), make(41), 1)
    check_norm(make(1, 40).expand(5, 40), make(40), make(40), 5)
    check_norm(make(2, 3, 4, 16), make(16), make(16), 1)
    check_norm(make(16), make(16), make(16), 1)
    check_norm(make(0, 16), make(16), make(16), 1)
    check_norm(torch.full((3, 64), 2.5, dtype=dtype, device=device), make(64), make(64), 1)


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_norm_far_from_zero(device):
    """The variance is taken around the mean: an offset of 1000 costs what it
    costs the inputs."""
    x = normal(seeded(), 3, 1000, device=device) + 1000
    check_norm(x, None, None, 1)


@pytest.mark.parametrize("device,dtype", PAIRS)
def test_norm_keeps_what_is_not_finite_in_its_group(device, dtype):
    x = normal(seeded(), 6, 96, dtype=dtype, device=device)
    clean = ops.layer_norm(x, groups=3)
    x[2, 40] = float("inf")
    y = ops.layer_norm(x, groups=3)
    assert not y[2, 32:64].isfinite().any()
    y[2, 32:64] = clean[2, 32:64]
    assert torch.equal(y, clean)


@pytest.mark.gpu
def test_norm_offsets_past_32_bits():
    x = torch.randn(300000, 8192, device="cuda", dtype=torch.bfloat16)
    y = ops.layer_norm(x)
    for rows in (slice(0, 4), slice(262140, 262148), slice(299996, 300000)):
        assert torch.equal(y[rows], ops.layer_norm(x[rows].clone()))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [4, 8])
def test_norm_rows_past_one_axis_of_a_launch(d):
    rows = (1 << 26) + 77
    x = torch.randn(rows, d, device="cuda", dtype=torch.float16)
    x.requires_grad_()
    y = ops.layer_norm(x)
    dx, = torch.autograd.grad(y, x, x.detach())
    for part in (slice(0, 5), slice((1 << 22) - 2, (1 << 22) + 2), slice(rows - 80, rows)):
        few = x.detach()[part].clone().requires_grad_()
        want = ops.layer_norm(few)
        assert torch.equal(y.detach()[part], want.detach())
        assert torch.equal(dx[part], torch.autograd.grad(want, few, few.detach())[0])


def test_norm_gradients_by_differences():
    gen = seeded()
    x, w, b = (normal(gen, *s).double().requires_grad_() for s in ((3, 12), (12,), (12,)))
    # the CPU form rounds nothing in 64 bits
    assert torch.autograd.gradcheck(lambda *t: ops.layer_norm(*t, groups=2), (x, w, b))


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_norm_refusals(device):
    x = torch.zeros(2, 12, device=device)
    with pytest.raises(ValueError, match="groups"):
        ops.layer_norm(x, groups=5)
    with pytest.raises(ValueError, match="groups"):
        ops.layer_norm(x[:, :0])
    with pytest.raises(ValueError, match="weight"):
        ops.layer_norm(x, torch.zeros(2, 6, device=device))
    with pytest.raises(ValueError, match="bias"):
        ops.layer_norm(x, None, torch.zeros(6, device=device))
    with pytest.raises(TypeError, match="float32"):
        ops.layer_norm(x, torch.zeros(12, device=device).half())
    if device == "cuda":
        with pytest.raises(TypeError, match="float32, bfloat16"):
            ops.layer_norm(x.double())
        with pytest.raises(ValueError, match="32768"):
            ops.layer_norm(torch.zeros(1, 32769, device=device))
        with pytest.raises(ValueError, match="different devices"):
            ops.layer_norm(x, torch.zeros(12))


# ---------------------------------------------------------------------------
# distill_loss
# ---------------------------------------------------------------------------
def exact_rows(x64, index, teacher, t):
    """The rows' losses, from the definition, row by row."""
    rows = []
    for n in range(x64.shape[0]):
        keep = [k for k in range(index.shape[1])
                if index[n, k] >= 0 and teacher[n, k] != -float("inf")]
        if not keep:
            rows.append(x64.new_zeros(()))
            continue
        log_p = torch.log_softmax(teacher[n, keep].double() / t, 0)
        log_q = torch.log_softmax(x64[n] / t, 0)[index[n, keep]]
        rows.append(t * t * (log_p.exp() * (log_p - log_q)).sum())
    return torch.stack(rows)


def check_distill(logits, index, teacher, t=1.0, reduction="mean", upstream=None, scale=1.0):
    leaf = logits.detach().requires_grad_()
    loss = ops.distill_loss(leaf, index, teacher, temperature=t, reduction=reduction, scale=scale)
    again = ops.distill_loss(logits.detach(), index, teacher, temperature=t, reduction=reduction,
                             scale=scale)
    assert torch.equal(loss.detach(), again) and loss.dtype == torch.float32
    v, top = logits.shape[-1], index.shape[-1]
    flat, i2, t2 = logits.detach().reshape(-1, v).cpu(), index.reshape(-1, top).cpu(), teacher.reshape(-1, top).cpu()
    x64 = flat.double().requires_grad_()
    rows = exact_rows(x64, i2, t2, t)
    some = ((i2 >= 0) & (t2 != -float("inf"))).any(1)
    count = max(1, int(some.sum())) if reduction == "mean" else 1
    want = rows if reduction == "none" else rows.sum() * (scale / count)
    g = torch.ones(()) if upstream is None else upstream
    grad, = torch.autograd.grad(loss, leaf, g.to(loss.device).expand_as(loss))
    dx, = torch.autograd.grad(want, x64, g.double().expand_as(want))
    # the log of the softmax's sum: each of the v terms' argument is off by a
    # few u of its size, the sum by at most v/128 + 64 additions
    s = x64.detach() / t
    lse = torch.logsumexp(torch.where(some[:, None], s, torch.zeros_like(s)), 1, keepdim=True)
    most = s.nan_to_num(0, 0, 0).abs().max(1, keepdim=True).values
    lse_off = U * (8 * most + 32 + v / 128)
    # slots: their masses off by the same kind of error over `top` terms
    tt = (t2.double() / t).nan_to_num(0, 0, 0).abs().max(1, keepdim=True).values
    p_off = U * (8 * tt + 32 + top)
    far = (2 * most + 2 * tt + 16)
    rows_off = (t * t * (lse_off + p_off * far + 8 * U * far)).squeeze(1) * some
    if reduction == "none":
        slack = rows_off
    else:
        slack = (rows_off.sum() + (len(rows) + 4) * U * rows.detach().abs().sum()) * abs(scale) / count
    within(loss.detach().cpu().reshape(want.shape), want.detach(), slack)
    q = (torch.where(some[:, None], s, torch.zeros_like(s)) - lse).exp() * some[:, None]
    each = (g.double().abs().expand(rows.shape) * t * abs(scale) / count)[:, None]
    # p's mass on a class is at most q + |dx| / each
    mass = q + dx.abs() / each.clamp_min(1e-300)
    slack = each * (q * (lse_off + 8 * U * (4 + (s.nan_to_num(0, 0, 0) - lse).abs())) + mass * (p_off + 8 * U))
    within(grad.cpu().reshape(-1, v), dx, slack)
    assert (grad.cpu().reshape(-1, v)[~some] == 0).all()


def distill_inputs(rows, v, top, dtype, device, seed=0, masked=0.0, itype=torch.int64):
    gen = seeded(seed)
    logits = normal(gen, rows, v, dtype=dtype, device=device, scale=3.0)
    index = torch.stack([torch.randperm(v, generator=gen)[:top] for _ in range(rows)])
    if masked:
        index = index.masked_fill(torch.rand(rows, top, generator=gen) < masked, -1)
    teacher = normal(gen, rows, top, dtype=dtype, device=device, scale=2.0)
    return logits, index.to(device=device, dtype=itype), teacher


@pytest.mark.parametrize("device,dtype", PAIRS)
@pytest.mark.parametrize("rows,v,top,t,reduction", [
    (1, 1, 1, 1.0, "mean"), (1, 2, 2, 2.0, "none"), (3, 21, 5, 1.5, "sum"), (20, 1000, 1, 1.0, "mean"),
    (7, 1001, 64, 2.0, "mean"), (5, 4097, 20, 4.0, "none"), (2, 33333, 100, 0.5, "mean"),
    (1, 70001, 1024, 1.0, "sum"), (1030, 4100, 300, 1.0, "mean"), (40, 4000, 1024, 1.0, "sum"), (70, 515, 70, 1.0, "mean"), (1030, 40, 3, 1.0, "mean")])
def test_distill(device, dtype, rows, v, top, t, reduction):
    check_distill(*distill_inputs(rows, v, top, dtype, device, seed=v), t, reduction)
    check_distill(*distill_inputs(rows, v, top, dtype, device, seed=v + 1, masked=0.4,
                                  itype=torch.int32), t, reduction)


@pytest.mark.parametrize("device,dtype", PAIRS)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_distill_masks_duplicates_and_extremes(device, dtype, reduction):
    logits, index, teacher = distill_inputs(8, 300, 6, dtype, device)
    low, inf = torch.finfo(dtype).min, float("inf")
    index[0] = -1                         # nothing left
    index[1, 1:] = -100                   # one slot
    index[2, 3] = index[2, 0]             # a class named twice
    index[3] = index[3, 0]                # one class six times
    teacher[4, 2:] = -inf                 # masked by its logit
    teacher[5] = -inf                     # all of them
    teacher[6, :3] = low                  # masses that vanish
    logits[7, ::2] = low                  # masked classes
    logits[7, index[7]] = 1.0
    logits[0, 7] = float("nan")           # never looked at
    logits[5] = inf
    check_distill(logits, index, teacher, 2.0, reduction)
    check_distill(logits, index, teacher, 2.0, reduction, upstream=torch.tensor(-0.37))
    if reduction == "none":
        check_distill(logits, index, teacher, 1.0, reduction, upstream=normal(seeded(5), 8))
    else:
        check_distill(logits, index, teacher, 2.0, reduction, scale=-1.75)
        check_distill(logits, index, teacher, 2.0, reduction, torch.tensor(3.0), scale=0.125)


@pytest.mark.parametrize("device,dtype", PAIRS)
@pytest.mark.parametrize("t", [0.5, 1.0, 3.0])
@pytest.mark.parametrize("v", [40, 9000])
def test_distill_row_of_the_lowest_value(device, dtype, t, v):
    """A row whose classes are all masked with the type's lowest value has a
    softmax all the same: they weigh alike, and the loss is log v."""
    logits, index, _ = distill_inputs(4, v, 1, dtype, device)
    logits[1] = torch.finfo(dtype).min
    logits[2] = -torch.finfo(dtype).min
    logits[3] = torch.finfo(dtype).min
    logits[3, v // 2:] = -float("inf")
    index[3] = 1
    leaf = logits.requires_grad_()
    rows = ops.distill_loss(leaf, index, temperature=t, reduction="none")
    want = t * t * torch.tensor([math.log(v), math.log(v), math.log(v // 2)], dtype=torch.float64,
                                device=device)
    # the sum of up to v ones is exact, its log and the product a few u off
    within(rows.detach()[1:], want, 16 * U * want)
    grad, = torch.autograd.grad(rows, leaf, torch.ones_like(rows))
    want = torch.full((4, v), t / v, dtype=torch.float64, device=device)
    want[3] = t / (v // 2)
    want[3, v // 2:] = 0
    want.scatter_add_(1, index, torch.full_like(want[:, :1], -t))
    within(grad[1:], want[1:], 16 * U * (want[1:].abs() + t / v))


@pytest.mark.parametrize("device,dtype", PAIRS)
def test_distill_class_that_is_masked_in_the_student(device, dtype):
    """-inf in the logits: no mass, and a loss of +inf where the teacher has some."""
    logits, index, teacher = distill_inputs(3, 50, 3, dtype, device)
    logits[0, 10:] = -float("inf")
    index[0] = torch.tensor([1, 2, 3], device=device)
    logits[1, index[1, 0]] = -float("inf")
    loss = ops.distill_loss(logits, index, teacher, reduction="none")
    assert loss[0].isfinite() and loss[1] == float("inf") and loss[2].isfinite()
    leaf = logits.clone().requires_grad_()
    ops.distill_loss(leaf, index, teacher, reduction="sum").backward()
    assert (leaf.grad[0, 10:] == 0).all() and leaf.grad[2].isfinite().all()


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_distill_bad_index_is_seen_and_stays_in_its_row(device):
    logits, index, teacher = distill_inputs(4, 50, 3, torch.float32, device)
    index[1, 2] = 50
    index[2, 0] = 2 ** 40
    leaf = logits.requires_grad_()
    loss = ops.distill_loss(leaf, index, teacher, reduction="none")
    assert loss.isnan().tolist() == [False, True, True, False]
    grad, = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
    assert grad.isnan().all(1).tolist() == [False, True, True, False]
    assert not grad[0].isnan().any() and not grad[3].isnan().any()


@pytest.mark.parametrize("device,dtype", PAIRS)
def test_distill_with_one_slot_is_cross_entropy(device, dtype):
    logits, index, teacher = distill_inputs(33, 1000, 1, dtype, device)
    index[4] = index[9] = -100
    ours = ops.distill_loss(logits, index, teacher)
    theirs = F.cross_entropy(logits.double(), index[:, 0])
    assert abs(float(ours) - float(theirs)) <= 200 * U * 30
    assert torch.equal(ours, ops.distill_loss(logits, index))
    alike = ops.distill_loss(logits, index.expand(33, 3))
    # three slots of a third each: sum_k 1/3 (log 1/3 - log q) = -log 3 - log q
    assert abs(float(alike) + math.log(3) - float(theirs)) <= 200 * U * 30


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_distill_strides_axes_and_empty(device):
    gen = seeded()
    logits, index, teacher = distill_inputs(12, 65, 4, torch.float32, device)
    check_distill(logits.view(3, 4, 65), index.view(3, 4, 4), teacher.view(3, 4, 4), 2.0, "none")
    check_distill(normal(gen, 12, 70, device=device)[:, 3:68], index, teacher)
    check_distill(logits.t().contiguous().t(), index.t().contiguous().t(), teacher.t().contiguous().t())
    check_distill(logits[:1].expand(12, 65), index[:1].expand(12, 4), teacher[:1].expand(12, 4))
    check_distill(logits[0], index[0], teacher[0])
    none = ops.distill_loss(logits[:0], index[:0], teacher[:0])
    assert float(none) == 0
    leaf = logits.detach().requires_grad_()
    ops.distill_loss(leaf, index[:, :0], teacher[:, :0]).backward()
    assert (leaf.grad == 0).all()


@pytest.mark.gpu
def test_distill_offsets_past_32_bits():
    v, rows = 150001, 16000
    logits = torch.randn(rows, v, device="cuda", dtype=torch.bfloat16)
    index = torch.randint(0, v, (rows, 8), device="cuda")
    teacher = torch.randn(rows, 8, device="cuda")
    few = [0, 1, 14316, 14317, 15999]
    leaf = logits.requires_grad_()
    loss = ops.distill_loss(leaf, index, teacher, reduction="none")
    grad, = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
    x64 = logits.detach()[few].double().requires_grad_()
    want = exact_rows(x64, index[few], teacher[few], 1.0)
    dx, = torch.autograd.grad(want.sum(), x64)
    within(loss.detach()[few], want.detach(), torch.full_like(want, U * (32 + v / 128 + 300)))
    within(grad[few], dx, U * 2000 * (dx.abs() + 1e-3))


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_distill_rows_past_one_axis_of_a_launch(reduction):
    rows, v = (1 << 26) + 77, 5
    logits = torch.randn(rows, v, device="cuda", dtype=torch.float16).requires_grad_()
    index = torch.randint(0, v, (rows, 1), device="cuda", dtype=torch.int32)
    loss = ops.distill_loss(logits, index, reduction=reduction)
    # an upstream gradient of other than 1 is written by the backward kernel
    dx, = torch.autograd.grad(loss, logits, torch.full_like(loss, 2.0))
    for part in (slice(0, 5), slice((1 << 24) - 3, (1 << 24) + 3), slice(rows - 80, rows)):
        few = logits.detach()[part].clone().requires_grad_()
        want = ops.distill_loss(few, index[part], reduction="none")
        if reduction == "none":
            assert torch.equal(loss.detach()[part], want.detach())
        assert torch.equal(dx[part], torch.autograd.grad(want, few, torch.full_like(want, 2.0))[0])


def test_distill_gradients_by_differences():
    logits, index, teacher = distill_inputs(4, 9, 3, torch.float32, "cpu", masked=0.3)
    x = logits.double().requires_grad_()
    for reduction in ("none", "sum", "mean"):
        assert torch.autograd.gradcheck(
            lambda x: ops.distill_loss(x, index, teacher, temperature=2.0, reduction=reduction), (x,))


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_distill_refusals(device):
    logits, index, teacher = distill_inputs(4, 9, 3, torch.float32, device)
    with pytest.raises(ValueError, match="reduction"):
        ops.distill_loss(logits, index, teacher, reduction="max")
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="temperature"):
            ops.distill_loss(logits, index, teacher, temperature=bad)
    for bad, how in ((2.0, "none"), (float("nan"), "mean"), (float("inf"), "sum")):
        with pytest.raises(ValueError, match="scale"):
            ops.distill_loss(logits, index, teacher, scale=bad, reduction=how)
    with pytest.raises(ValueError, match="does not fit"):
        ops.distill_loss(logits, index[:, :2], teacher)
    with pytest.raises(ValueError, match="does not fit"):
        ops.distill_loss(logits[:3], index, teacher)
    with pytest.raises(ValueError, match="no classes"):
        ops.distill_loss(logits[:, :0], index, teacher)
    with pytest.raises(TypeError, match="index"):
        ops.distill_loss(logits, index.float(), teacher)
    with pytest.raises(TypeError, match="floats"):
        ops.distill_loss(logits.long(), index, teacher)
    with pytest.raises(ValueError, match="teacher"):
        ops.distill_loss(logits, index, teacher.requires_grad_())
    with pytest.raises(ValueError, match="1024"):
        wide = torch.zeros(4, 1025, device=device)
        ops.distill_loss(logits, wide.long(), wide)
    if device == "cuda":
        with pytest.raises(TypeError, match="float32, bfloat16"):
            ops.distill_loss(logits.double(), index, teacher.detach())
        with pytest.raises(ValueError, match="different devices"):
            ops.distill_loss(logits, index.cpu(), teacher.detach())


# ---------------------------------------------------------------------------
# together, and as a program uses them
# ---------------------------------------------------------------------------
def head(x, nw, nb, w, b, r, index, teacher):
    h = ops.layer_norm(x, nw, nb)
    return ops.distill_loss(ops.linear(h, w, b, activation="gelu", residual=r), index, teacher,
                            temperature=2.0)


def head_inputs(device, dtype, rows=37, width=96, v=530, top=5):
    gen = seeded(11)
    make = lambda *s, scale=1.0: normal(gen, *s, dtype=dtype, device=device, scale=scale)  # noqa: E731
    leaves = [make(rows, width), make(width), make(width), make(v, width, scale=0.1), make(v), make(rows, v)]
    index = torch.stack([torch.randperm(v, generator=gen)[:top] for _ in range(rows)]).to(device)
    return [t.requires_grad_() for t in leaves], index, make(rows, top)


@pytest.mark.parametrize("device,dtype", PAIRS)
def test_head_together(device, dtype):
    """Normalise, project, take the loss, and all gradients."""
    leaves, index, teacher = head_inputs(device, dtype)
    loss = head(*leaves, index, teacher)
    grads = torch.autograd.grad(loss, leaves)
    exact = [t.detach().double().cpu().requires_grad_() for t in leaves]
    x, nw, nb, w, b, r = exact
    y = F.gelu(F.linear(F.layer_norm(x, (x.shape[1],), nw, nb), w, b)) + r
    want = exact_rows(y, index.cpu(), teacher.cpu(), 2.0).mean()
    # three stored tensors lie between the inputs and the loss: of its
    # gradients, relative to their length, a few half steps
    step = half_step(dtype)
    assert abs(float(loss) - float(want)) <= 8 * (step + 100 * U) * float(want)
    for ours, theirs in zip(grads, torch.autograd.grad(want, exact)):
        off = (ours.double().cpu() - theirs).norm() / theirs.norm()
        assert off <= 8 * step + 400 * U, off


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_head_is_the_same_every_time_and_on_another_stream(dtype):
    leaves, index, teacher = head_inputs("cuda", dtype, rows=300, width=1000, v=5001)
    first = torch.autograd.grad(head(*leaves, index, teacher), leaves)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = torch.autograd.grad(head(*leaves, index, teacher), leaves)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, other):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_head_captured_and_replayed():
    """Forward and backward in a graph, new inputs between the replays, eager
    work beside them, and a second graph that shares nothing with the first."""
    leaves, index, teacher = head_inputs("cuda", torch.bfloat16, rows=40, width=512, v=5000)

    def step():
        loss = head(*leaves, index, teacher)
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for seed in range(4):
        gen = seeded(seed)
        with torch.no_grad():
            leaves[0].copy_(normal(gen, 40, 512))
            index.copy_(torch.randint(0, 5000, (40, 5), generator=gen))
        want = step()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_head_second_derivative(device):
    leaves, index, teacher = head_inputs(device, torch.float32, rows=5, width=12, v=20, top=3)

    def penalty(leaves, index, teacher):
        grads = torch.autograd.grad(head(*leaves, index, teacher), leaves, create_graph=True)
        return torch.autograd.grad(sum((g * g).sum() for g in grads), leaves)

    ours = penalty(leaves, index, teacher)
    exact = penalty([t.detach().double().cpu().requires_grad_() for t in leaves], index.cpu(),
                    teacher.double().cpu())
    for a, b in zip(ours, exact):
        assert (a.double().cpu() - b).norm() <= 2000 * U * b.norm()


@pytest.mark.gpu
def test_autocast_casts_as_torch_does():
    x, w = torch.randn(6, 64, device="cuda"), torch.randn(32, 64, device="cuda", requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = ops.linear(x, w, torch.zeros(32, device="cuda"))
        assert y.dtype == torch.bfloat16 == F.linear(x, w).dtype
        assert ops.layer_norm(y).dtype == torch.float32
    y.float().sum().backward()
    assert w.grad.dtype == torch.float32


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_results_may_be_changed_in_place(device):
    x, w = normal(seeded(), 2, 3, 8, device=device), normal(seeded(1), 6, 8, device=device)
    for act, residual in (("none", False), ("gelu", True)):
        r = torch.ones(2, 3, 6, device=device) if residual else None
        lead, flat = x.clone().requires_grad_(), x.flatten(0, 1).requires_grad_()
        y = ops.linear(lead, w, activation=act, residual=r).mul_(2)
        z = ops.linear(flat, w, activation=act, residual=None if r is None else r.flatten(0, 1)) * 2
        assert torch.equal(y.flatten(0, 1), z)
        y.sum().backward(), z.sum().backward()
        assert torch.equal(lead.grad.flatten(0, 1), flat.grad)
    lead = x.clone().requires_grad_()
    ops.layer_norm(lead).mul_(2).sum().backward()


def test_tensors_without_data():
    x = torch.empty(3, 8, device="meta", requires_grad=True)
    y = ops.linear(x, torch.empty(5, 8, device="meta"), activation="gelu")
    assert y.shape == (3, 5) and y.device.type == "meta"
    assert ops.layer_norm(x, groups=2).shape == (3, 8)
    loss = ops.distill_loss(x, torch.empty(3, 2, dtype=torch.long, device="meta"))
    assert torch.autograd.grad(loss, x)[0].shape == (3, 8)


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_sign_that_is_still_to_be_turned(device):
    turned = torch.randn(4, 8, 2, device=device).view(4, 16)
    turned = torch.view_as_complex(turned.view(4, 8, 2)).conj().imag
    assert turned.is_neg()
    plain = turned.resolve_neg()
    w = torch.randn(6, 8, device=device)
    index = torch.zeros(4, 1, dtype=torch.long, device=device)
    bound = 64 * U  # a sum of 8 terms of ordinary size, either way
    for f in (lambda t: ops.linear(t, w), ops.layer_norm,
              lambda t: ops.distill_loss(t, index, reduction="none")):
        assert (f(turned) - f(plain)).abs().max() <= bound
    for f in (lambda t: ops.linear(t, w), ops.layer_norm):
        x = plain.clone().requires_grad_()
        y = f(x)
        up = torch.view_as_complex(torch.randn(*y.shape, 2, device=device)).conj().imag
        a, = torch.autograd.grad(y, x, up, retain_graph=True)
        b, = torch.autograd.grad(y, x, up.resolve_neg())
        assert torch.equal(a, b)


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_forward_mode_runs_the_formula(device):
    x, v = (torch.randn(3, 8, device=device) for _ in range(2))
    w = torch.randn(6, 8, device=device)
    index = torch.zeros(3, 1, dtype=torch.long, device=device)
    for f in (lambda t: ops.linear(t, w, activation="silu"), ops.layer_norm,
              lambda t: ops.distill_loss(t, index)):
        with torch.autograd.forward_ad.dual_level():
            y = f(torch.autograd.forward_ad.make_dual(x, v))
            got = torch.autograd.forward_ad.unpack_dual(y).tangent
        assert got is not None
        leaf = x.clone().requires_grad_()
        z = f(leaf)
        up = torch.randn_like(z)
        back, = torch.autograd.grad(z, leaf, up)
        # both are up^T J v: sums of fewer than 32 terms of ordinary size
        assert abs((got * up).sum() - (back * v).sum()) <= 1e-3


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_compiled_calls_run_the_formula(device):
    x, w = torch.randn(6, 8, device=device), torch.randn(5, 8, device=device)
    index = torch.zeros(6, 1, dtype=torch.long, device=device)

    def f(x):
        return ops.linear(x, w, activation="gelu"), ops.layer_norm(x), ops.distill_loss(x, index)

    for got, want in zip(torch.compile(f, backend="eager", fullgraph=True)(x), f(x)):
        assert (got - want).abs().max() <= 64 * U


CAPTURED_FIRST = """
import torch
from k8s_device_plugin_amd import ops
x, w = torch.randn(5, 64, device="cuda"), torch.randn(40, 64, device="cuda")
index = torch.zeros(5, 1, dtype=torch.long, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = ops.layer_norm(ops.linear(x, w))
    loss = ops.distill_loss(y, index)
for _ in range(3):
    x.normal_()
    graph.replay()
    want = ops.layer_norm(ops.linear(x, w))
    assert torch.equal(y, want) and torch.equal(loss, ops.distill_loss(want, index))
    torch.cuda.synchronize()
print("same")
"""


@pytest.mark.gpu
def test_first_call_of_a_process_may_be_captured():
    out = subprocess.run([sys.executable, "-c", CAPTURED_FIRST], cwd=REPO, capture_output=True,
                         text=True, timeout=100)
    assert out.returncode == 0 and "same" in out.stdout, out.stderr[-2000:]


@pytest.mark.gpu
def test_traced_and_transformed_calls_run_the_formula():
    x, w = torch.randn(6, 64, device="cuda"), torch.randn(32, 64, device="cuda")
    y = ops.linear(x, w)
    mapped = torch.func.vmap(lambda r: ops.linear(r, w))(x)
    traced = torch.jit.trace(lambda r: ops.linear(r, w), (x,))(x)
    for other in (mapped, traced):
        assert (y - other).abs().max() <= 66 * 2 * U * float((x.abs() @ w.abs().t()).max())


def test_bad_calls_of_the_library_are_refused():
    """The C entry points look at what they are given before they launch."""
    import ctypes

    from k8s_device_plugin_amd.ops import _native as n

    lib = n.library()
    at = torch.zeros(64, 64).data_ptr()

    def linear(**how):
        a = dict(x=at, w=at, y=at, m=4, n=4, k=4, xs0=4, xs1=1, ws0=4, ws1=1, dtype=0, act=0)
        return lib.vgpu_ops_linear(ctypes.byref(n.LinearArgs(**{**a, **how})), None)

    for how in (dict(m=0), dict(n=-1), dict(k=0), dict(dtype=3), dict(act=4), dict(xs0=-4),
                dict(y=None), dict(w=None), dict(dy=at, act=1), dict(xs1=2)):
        assert linear(**how) < 0, how  # the last: a workspace is wanted

    def norm(**how):
        a = dict(x=at, y=at, ldx=8, ldy=8, rows=2, groups=1, d=8, eps=1e-5)
        return lib.vgpu_ops_norm(ctypes.byref(n.NormArgs(**{**a, **how})), None)

    for how in (dict(rows=0), dict(d=0), dict(d=32769), dict(groups=0), dict(dtype=7), dict(wtype=2),
                dict(y=None), dict(dy=at, parts=0), dict(dy=at, parts=2, dweight=at)):
        assert norm(**how) < 0, how

    def distill(**how):
        a = dict(x=at, index=at, rows_loss=at, state=at, origin=at, loss=at, counts=at, ldx=8, ldi=1,
                 rows=2, v=8, top=1, index_bytes=8, chunks=1, reduction=2, temperature=1.0, scale=1.0)
        return lib.vgpu_ops_distill(ctypes.byref(n.DistillArgs(**{**a, **how})), None)

    for how in (dict(rows=0), dict(v=0), dict(top=0), dict(top=1025), dict(chunks=0), dict(dtype=9),
                dict(index_bytes=2), dict(reduction=3), dict(temperature=0.0), dict(state=None),
                dict(counts=None), dict(loss=None), dict(chunks=2), dict(dx=at), dict(grad=at)):
        assert distill(**how) < 0, how


@pytest.mark.gpu
def test_two_threads_at_once():
    """Calls from two threads on two streams share no state."""
    import threading

    leaves, index, teacher = head_inputs("cuda", torch.float32, rows=20, width=2048, v=1000)
    want = torch.autograd.grad(head(*leaves, index, teacher), leaves)
    torch.cuda.synchronize()
    wrong = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = torch.autograd.grad(head(*leaves, index, teacher), leaves)
                torch.cuda.current_stream().synchronize()
                wrong.extend(i for i, (a, b) in enumerate(zip(got, want)) if not torch.equal(a, b))

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_control_plane_needs_no_torch():
    code = ("import sys; sys.modules['torch'] = None\n"
            "from k8s_device_plugin_amd import ops\n"
            "assert ops.cus_for_percent(50) == 128\n"
            "try: ops.linear\n"
            "except ImportError: print('ok')\n")
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=REPO)
    assert out.stdout.strip() == "ok", out.stderr
    with pytest.raises(AttributeError, match="matmul_nothing"):
        ops.matmul_nothing


def test_missing_library_is_an_error(monkeypatch, tmp_path):
    from k8s_device_plugin_amd.ops import _native

    monkeypatch.setattr(_native, "PACKAGE", tmp_path / "package")
    _native.library.cache_clear()
    with pytest.raises(RuntimeError, match="make native"):
        _native.library()
    _native.library.cache_clear()


@pytest.mark.parametrize("device,dtype", PAIRS)
@pytest.mark.parametrize("rows,v", [(20, 1000), (600, 9001)])
def test_distill_backward_twice(device, dtype, rows, v):
    """The gradient that a first backward pass hands out is the caller's: a
    second pass does not see what was done to it."""
    logits, index, teacher = distill_inputs(rows, v, 3, dtype, device)
    leaf = logits.requires_grad_()
    loss = ops.distill_loss(leaf, index, teacher, temperature=2.0)
    first, = torch.autograd.grad(loss, leaf, retain_graph=True)
    kept = first.clone()
    first.mul_(7)
    second, = torch.autograd.grad(loss, leaf, retain_graph=True)
    assert torch.equal(second, kept)
    leaf.grad = None
    loss.backward(retain_graph=True)
    loss.backward()
    assert torch.equal(leaf.grad, kept + kept)
