"""Cases for the operators of a model's head: normalise, project, take the loss.

``run`` computes each in its plain form (elementary torch operations in 32
bits, rounded once at the end) or, where ``own`` is true, through this
package's public entry points.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}

# The largest listed product (8192 x 4096 x 16384) and the largest listed
# normalisation and loss bound what draw() may give.
MOST_FLOPS = 2 * 8192 * 4096 * 16384
MOST_NORM = 16384 * 8192
MOST_LOGITS = 4096 * 131072


def listed():
    return [
        # one token through a square projection while serving: latency
        {"name": "linear_one_token", "op": "linear", "dtype": "bf16", "m": 1, "k": 4096, "n": 4096,
         "act": "silu", "bias": True, "residual": True, "train": False, "pad": 0},
        # VGG-16's first classifier layer at the serving batch: streams 411 MB of weights
        {"name": "linear_vgg_serving", "op": "linear", "dtype": "fp32", "m": 20, "k": 25088, "n": 4096,
         "act": "relu", "bias": True, "residual": False, "train": False, "pad": 0},
        # the same layer in a training step at the zoo's batch of 2
        {"name": "linear_vgg_training", "op": "linear", "dtype": "fp32", "m": 2, "k": 25088, "n": 4096,
         "act": "relu", "bias": True, "residual": False, "train": True, "pad": 0},
        # a prompt's tokens through the first projection of a feed-forward block: the matrix cores
        {"name": "linear_many_tokens", "op": "linear", "dtype": "bf16", "m": 8192, "k": 4096, "n": 16384,
         "act": "gelu", "bias": True, "residual": False, "train": False, "pad": 0},
        # a training step of a projection with a residual, an odd number of tokens
        {"name": "linear_training", "op": "linear", "dtype": "fp16", "m": 4099, "k": 4096, "n": 10240,
         "act": "gelu", "bias": True, "residual": True, "train": True, "pad": 8},
        # DeepLab's pooled branch: 32 groups of 8 channels of a 1x1 map, batch 2
        {"name": "norm_pooled_groups", "op": "norm", "dtype": "fp32", "rows": 2, "groups": 32, "d": 8,
         "train": True, "pad": 0},
        # one token's normalisation while serving
        {"name": "norm_one_token", "op": "norm", "dtype": "bf16", "rows": 1, "groups": 1, "d": 4096,
         "train": False, "pad": 0},
        # rows of an odd width out of a wider buffer
        {"name": "norm_odd_rows", "op": "norm", "dtype": "fp16", "rows": 2049, "groups": 1, "d": 5001,
         "train": True, "pad": 7},
        # a training step over a large batch of tokens
        {"name": "norm_training", "op": "norm", "dtype": "bf16", "rows": 16384, "groups": 1, "d": 8192,
         "train": True, "pad": 0},
        # the zoo's training loss: 20 images, 1000 classes, a label each
        {"name": "loss_labels", "op": "loss", "dtype": "fp32", "rows": 20, "v": 1000, "top": 1,
         "temperature": 1.0, "train": True, "masked": False},
        # scoring a few sequences' last tokens against a teacher, forward only
        {"name": "loss_few_rows", "op": "loss", "dtype": "fp16", "rows": 5, "v": 150001, "top": 20,
         "temperature": 1.5, "train": False, "masked": True},
        # a distillation step over a large vocabulary, some tokens without a target
        {"name": "loss_vocabulary", "op": "loss", "dtype": "bf16", "rows": 4096, "v": 131072, "top": 64,
         "temperature": 2.0, "train": True, "masked": True},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["linear", "norm", "loss"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    train = rng.random() < 0.5
    if op == "linear":
        m, k, n = _spread(rng, 1, 8192), _spread(rng, 16, 25088), _spread(rng, 16, 16384)
        if rng.random() < 0.5:  # widths are multiples of 8 as often as not
            k, n = (k + 7) // 8 * 8, (n + 7) // 8 * 8
        m = max(1, min(m, MOST_FLOPS // ((6 if train else 2) * k * n)))
        return {"op": op, "dtype": dtype, "m": m, "k": k, "n": n,
                "act": rng.choice(["none", "relu", "gelu", "silu"]), "bias": rng.random() < 0.7,
                "residual": rng.random() < 0.5, "train": train, "pad": rng.choice([0, 0, 8, 3])}
    if op == "norm":
        rows, groups, d = _spread(rng, 1, 16384), rng.choice([1, 1, 1, 32]), _spread(rng, 8, 16384)
        d = max(8, d // groups)
        rows = max(1, min(rows, MOST_NORM // (groups * d)))
        return {"op": op, "dtype": dtype, "rows": rows, "groups": groups, "d": d,
                "train": train, "pad": rng.choice([0, 0, 8, 7])}
    rows, v = _spread(rng, 1, 4096), _spread(rng, 21, 151000)
    rows = max(1, min(rows, MOST_LOGITS // v // (2 if dtype == "fp32" else 1)))
    return {"op": op, "dtype": dtype, "rows": rows, "v": v, "top": min(v, _spread(rng, 1, 64)),
            "temperature": rng.choice([1.0, 1.5, 2.0, 4.0]), "train": train, "masked": rng.random() < 0.5}


def work(case):
    size = SIZES[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        elements = m * k + n * k + m * n + n * case["bias"] + m * n * case["residual"]
        if case["train"]:  # the gradient comes in; those of x, weight and bias go out
            elements += m * n + m * k + n * k + n * case["bias"]
        return {"bytes": elements * size, "flops": (6 if case["train"] else 2) * m * n * k}
    if case["op"] == "norm":
        count, width = case["rows"] * case["groups"] * case["d"], case["groups"] * case["d"]
        if case["train"]:
            return {"bytes": (4 * count + 4 * width) * size, "flops": 20 * count}
        return {"bytes": (2 * count + 2 * width) * size, "flops": 8 * count}
    count, slots = case["rows"] * case["v"], case["rows"] * case["top"]
    return {"bytes": count * size * (2 if case["train"] else 1) + slots * (8 + size) + 4,
            "flops": count * (8 if case["train"] else 4)}


def _rows(shape, pad, make):
    """A matrix whose rows stand ``pad`` elements apart in a wider buffer."""
    rows, width = shape
    return make(rows, width + pad)[:, :width]


def prepare(case, seed):
    dtype = DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, shift=0.0, to=dtype):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale).add_(shift).to(to)

    state = {"case": case}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        state["x"] = _rows((m, k), case["pad"], normal)
        state["weight"] = normal(n, k, scale=k ** -0.5)
        state["bias"] = normal(n, scale=0.1) if case["bias"] else None
        state["residual"] = normal(m, n) if case["residual"] else None
        state["grad"] = normal(m, n) if case["train"] else None
        leaves = ("x", "weight", "bias", "residual")
    elif case["op"] == "norm":
        rows, width = case["rows"], case["groups"] * case["d"]
        state["x"] = _rows((rows, width), case["pad"], lambda *s: normal(*s, scale=1.5, shift=0.5))
        state["weight"] = normal(width, scale=0.1, shift=1.0)
        state["bias"] = normal(width, scale=0.1)
        state["grad"] = normal(rows, width) if case["train"] else None
        leaves = ("x", "weight", "bias")
    else:
        rows, v, top = case["rows"], case["v"], case["top"]
        state["logits"] = normal(rows, v, scale=2.0)
        state["teacher"] = normal(rows, top, scale=2.0).sort(dim=1, descending=True).values
        # distinct classes of a row: a random start, then steps that never meet it again
        start = torch.randint(0, v, (rows, 1), generator=gen, device="cuda")
        index = (start + torch.arange(top, device="cuda") * max(1, v // top)) % v
        if case["masked"]:  # a tenth of the slots, and every seventh row whole
            gone = torch.rand(rows, top, generator=gen, device="cuda") < 0.1
            gone[3::7] = True
            index = index.masked_fill(gone, -1)
        state["index"] = index
        leaves = ("logits",)
    if case["train"]:
        for name in leaves:
            if state[name] is not None:
                state[name] = state[name].detach().requires_grad_()
    return state


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _activate(z, act):
    """The activation and its derivative."""
    if act == "none":
        return z, None
    if act == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))


def _plain_linear(s):
    case, dtype = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y, slope = _activate(z, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(dtype)}
    if case["train"]:
        dz = s["grad"].float()
        if slope is not None:
            dz = dz * slope
        out["x"] = (dz @ w).to(dtype)
        out["weight"] = (dz.t() @ x).to(dtype)
        if s["bias"] is not None:
            out["bias"] = dz.sum(0).to(dtype)
        if s["residual"] is not None:
            out["residual"] = s["grad"]
    return out


def _plain_norm(s):
    case, dtype = s["case"], s["x"].dtype
    shape = (case["rows"], case["groups"], case["d"])
    x = s["x"].float().reshape(shape)
    w = s["weight"].float().reshape(shape[1:])
    mean = x.mean(-1, keepdim=True)
    centred = x - mean
    scale = 1 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + 1e-5)
    h = centred * scale
    y = h * w + s["bias"].float().reshape(shape[1:])
    out = {"y": y.flatten(1).to(dtype)}
    if case["train"]:
        g = s["grad"].float().reshape(shape)
        a = g * w
        dx = (a - a.mean(-1, keepdim=True) - h * (a * h).mean(-1, keepdim=True)) * scale
        out["x"] = dx.flatten(1).to(dtype)
        out["weight"] = (g * h).sum(0).flatten().to(dtype)
        out["bias"] = g.sum(0).flatten().to(dtype)
    return out


def _plain_loss(s):
    case, t = s["case"], s["case"]["temperature"]
    x = s["logits"].float() / t
    top = x.max(1, keepdim=True).values
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    here = s["index"] >= 0
    index = s["index"].clamp_min(0)
    teach = (s["teacher"].float() / t).masked_fill(~here, -math.inf)
    some = here.any(1, keepdim=True)
    high = teach.max(1, keepdim=True).values.masked_fill(~some, 0)
    p = torch.exp(teach - high)
    mass = p.sum(1, keepdim=True).clamp_min(1e-30)
    p = p / mass
    log_p = (teach - high - torch.log(mass)).masked_fill(~here, 0)
    log_q = x.gather(1, index) - top - torch.log(total)
    rows = t * t * (p * (log_p - log_q)).sum(1)
    if not case["train"]:
        return {"rows": rows}
    count = some.sum().clamp_min(1)
    grad = (e / total).scatter_add(1, index, -p) * (some * t / count)
    return {"loss": rows.sum() / count, "logits": grad.to(s["logits"].dtype)}


# ---------------------------------------------------------------------------
# The package's own
# ---------------------------------------------------------------------------
def _gradients(s, y, grad, names):
    names = [n for n in names if s[n] is not None]
    return dict(zip(names, torch.autograd.grad(y, [s[n] for n in names], grad)))


def _own(s):
    from k8s_device_plugin_amd import ops

    case = s["case"]
    if case["op"] == "linear":
        y = ops.linear(s["x"], s["weight"], s["bias"], activation=case["act"], residual=s["residual"])
        names = ("x", "weight", "bias", "residual")
    elif case["op"] == "norm":
        y = ops.layer_norm(s["x"], s["weight"], s["bias"], groups=case["groups"])
        names = ("x", "weight", "bias")
    else:
        loss = ops.distill_loss(s["logits"], s["index"], s["teacher"], temperature=case["temperature"],
                                reduction="mean" if case["train"] else "none")
        if not case["train"]:
            return {"rows": loss}
        return {"loss": loss.detach(), **_gradients(s, loss, None, ("logits",))}
    if not case["train"]:
        return {"y": y}
    return {"y": y.detach(), **_gradients(s, y, s["grad"], names)}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"linear": _plain_linear, "norm": _plain_norm, "loss": _plain_loss}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# In 64 bits, by differentiating the definition
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    leaf = {n: v.detach().double().requires_grad_(case["train"])
            for n, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if case["op"] == "linear":
        z = torch.nn.functional.linear(leaf["x"], leaf["weight"], leaf.get("bias"))
        f = {"none": lambda u: u, "relu": torch.relu, "silu": torch.nn.functional.silu,
             "gelu": torch.nn.functional.gelu}[case["act"]]
        y = f(z) if s["residual"] is None else f(z) + leaf["residual"]
        names = [n for n in ("x", "weight", "bias", "residual") if n in leaf]
    elif case["op"] == "norm":
        split = leaf["x"].unflatten(1, (case["groups"], case["d"]))
        var, mean = torch.var_mean(split, -1, correction=0, keepdim=True)
        y = ((split - mean) * (var + 1e-5).rsqrt()).flatten(1) * leaf["weight"] + leaf["bias"]
        names = ["x", "weight", "bias"]
    else:
        t, index = case["temperature"], s["index"]
        log_q = torch.log_softmax(leaf["logits"] / t, 1)
        rows = []
        for n in range(case["rows"]):  # row by row: only the slots that are there
            k = (index[n] >= 0).nonzero()[:, 0]
            if len(k) == 0:
                rows.append(leaf["logits"].new_zeros(()))
                continue
            log_p = torch.log_softmax(leaf["teacher"][n, k].detach() / t, 0)
            rows.append(t * t * (log_p.exp() * (log_p - log_q[n, index[n, k]])).sum())
        rows = torch.stack(rows)
        if not case["train"]:
            return {"rows": rows.detach()}
        y = rows.sum() / max(1, int((index >= 0).any(1).sum()))
        return {"loss": y.detach(), "logits": torch.autograd.grad(y, leaf["logits"])[0]}
    if not case["train"]:
        return {"y": y.detach()}
    grads = torch.autograd.grad(y, [leaf[n] for n in names], leaf["grad"])
    return {"y": y.detach(), **dict(zip(names, grads))}
