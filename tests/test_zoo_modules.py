"""The layers of the zoo's heads stay torch's modules: what is hung on them,
put in their place or made of them works as it does on any other."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from k8s_device_plugin_amd.models import zoo
from test_zoo_heads import GPU, close


def pooled_inputs(device):
    torch.manual_seed(0)
    return zoo.ASPP(64).to(device), torch.randn(2, 64, 5, 7, device=device)


@pytest.fixture
def calls(monkeypatch):
    """The operators' calls out of the zoo."""
    seen = []
    for name in ("linear", "layer_norm"):
        f = getattr(zoo.ops, name)
        monkeypatch.setattr(zoo.ops, name, lambda *a, f=f, name=name, **k: (seen.append(name), f(*a, **k))[1],
                            raising=False)
    return seen


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_heads_take_the_kernels_on_a_gpu(device, calls):
    on = device == "cuda"
    aspp, x = pooled_inputs(device)
    aspp.pooled(x)
    assert calls == (["linear", "layer_norm"] if on else [])
    zoo.LSTMNet(8, 16, 1).to(device)(torch.randn(2, 3, 8, device=device))
    zoo.VGG16().classifier.to(device)(torch.randn(2, 25088, device=device))
    assert calls == (["linear", "layer_norm", *["linear"] * 4] if on else [])


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("kind", ["forward", "before", "backward"])
def test_hooks_on_the_heads_layers_run(device, kind):
    aspp, x = pooled_inputs(device)
    head, lstm = zoo.VGG16().classifier.to(device), zoo.LSTMNet(8, 16, 1).to(device)
    x.requires_grad_()  # a layer without parameters has a gradient to pass on
    fired = []
    layers = [("aspp", m) for m in (aspp.gp, *aspp.gp)] + [("vgg", m) for m in (head, *head)] + [
        ("lstm", lstm.fc)]
    for name, m in layers:
        note = lambda m, *_: fired.append(m)  # noqa: E731
        {"forward": m.register_forward_hook, "before": m.register_forward_pre_hook,
         "backward": m.register_full_backward_hook}[kind](note)
        for part in m.modules():
            if hasattr(part, "inplace"):
                part.inplace = False  # a backward hook's output may not be changed
    loss = (aspp.pooled(x).sum() + head(torch.randn(2, 25088, device=device)).sum()
            + lstm(torch.randn(2, 3, 8, device=device)).sum())
    loss.backward()
    for name, m in layers:
        assert fired.count(m) == 1, (name, m)


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_heads_layers_may_be_pruned_normalised_and_replaced(device):
    from torch.nn.utils import parametrizations, prune, spectral_norm

    def steps(model, x, parameters):
        opt = torch.optim.SGD(parameters, lr=0.1)
        for _ in range(3):
            opt.zero_grad()
            (model(x) ** 2).sum().backward()
            opt.step()

    for way in ("prune", "spectral", "parametrized", "replaced"):
        aspp, x = pooled_inputs(device)
        lstm, z = zoo.LSTMNet(8, 16, 1).to(device), torch.randn(2, 3, 8, device=device)
        for holder, key, model, data in ((aspp.gp, "1", aspp.pooled, x), (lstm, "fc", lstm, z)):
            layer = getattr(holder, key)
            if way == "prune":
                prune.l1_unstructured(layer, "weight", 0.5)
            elif way == "spectral":
                spectral_norm(layer)
            elif way == "parametrized":
                parametrizations.spectral_norm(layer)
            else:
                setattr(holder, key, nn.Sequential(layer, nn.Tanh()).to(device))
            learnt = list(getattr(holder, key).parameters())
            before = [p.detach().clone() for p in learnt]
            steps(model, data, learnt)
            assert not torch.equal(before[0], learnt[0]), (way, key)
            if way == "prune":
                layer = getattr(holder, key)
                assert (layer.weight[layer.weight_mask == 0] == 0).all()
        if way == "replaced":
            assert lstm(z).abs().max() <= 1
        aspp.gp[2] = nn.Identity()
        assert aspp.pooled(x).shape == (2, 256, 1, 1)
        aspp.gp = nn.Identity()
        assert aspp.pooled(x).shape == x.shape


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_heads_trace_symbolically(device):
    aspp, x = pooled_inputs(device)
    z = torch.randn(2, 3, 8, device=device)
    head = zoo.VGG16().classifier
    for model, data in ((aspp.eval(), x), (zoo.LSTMNet(8, 16, 1).to(device), z),
                        (zoo.Classifier(*head[3:]).eval().to(device), torch.randn(2, 4096, device=device))):
        traced = torch.fx.symbolic_trace(model)
        assert close(traced(data), model(data))
    names = [n.target for n in torch.fx.symbolic_trace(zoo.Classifier(*head)).graph.nodes
             if n.op == "call_module"]
    assert names == [str(i) for i in range(7)]


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_heads_compile_and_script_whole(device):
    aspp, x = pooled_inputs(device)
    aspp = aspp.eval()
    lstm, z = zoo.LSTMNet(8, 16, 1).to(device), torch.randn(2, 3, 8, device=device)
    head = zoo.Classifier(nn.Linear(8, 12), nn.ReLU(inplace=True), nn.Linear(12, 5)).to(device)
    v = torch.randn(2, 8, device=device)
    for model, data in ((aspp, x), (lstm, z), (head, v)):
        assert close(torch.jit.script(model)(data), model(data))
    for model, data in ((aspp, x), (head, v)):
        assert close(torch.compile(model, backend="eager", fullgraph=True)(data), model(data))


def test_heads_may_be_quantised():
    lstm = zoo.LSTMNet(8, 16, 1)
    head = zoo.VGG16().classifier
    for model in (lstm, zoo.Classifier(*head[3:])):
        small = torch.ao.quantization.quantize_dynamic(model, {nn.Linear})
        assert not any(type(m) is nn.Linear for m in small.modules())
        assert any("Quantized" in type(m).__name__ or "quantized" in type(m).__module__
                   for m in small.modules())
    x = torch.randn(2, 4096)
    off = (small.eval()(x) - zoo.Classifier(*head[3:]).eval()(x)).norm()
    # 8 bits a value, weights and inputs, through two layers: half a step of 127
    # or 255 levels of each, against sums of many terms of either sign
    assert off <= 0.1 * small(x).norm()


@pytest.mark.gpu
def test_heads_leave_to_torch_what_the_operators_refuse():
    fc = nn.Linear(8, 4).cuda()
    with pytest.raises(RuntimeError):
        zoo.project(fc, torch.randn(2, 8, device="cuda").half())
    assert zoo.project(fc.double(), torch.randn(2, 8, device="cuda").double()).dtype == torch.float64
    wide = nn.Linear(1 << 21, 2).cuda()
    assert zoo.project(wide, torch.randn(2, 1 << 21, device="cuda")).shape == (2, 2)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert zoo.project(fc.float(), torch.randn(2, 8, device="cuda")).dtype == torch.bfloat16


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_loss_takes_every_target_of_cross_entropy(device):
    case = zoo.CASES["resnet50_train"]
    gen = torch.Generator().manual_seed(0)
    out = torch.randn(6, 9, generator=gen).to(device)
    maps = torch.randn(6, 9, 4, generator=gen).to(device)
    label = torch.randint(0, 9, (6,), generator=gen).to(device)
    ignored = label.clone()
    ignored[2] = -100
    for logits, y in ((out, torch.softmax(out + 1, 1)), (maps, label[:, None].expand(6, 4)),
                      (maps, torch.softmax(maps + 1, 1)), (out[0], label[0]),
                      (out.double(), label), (out, label), (out, ignored)):
        a, b = (logits.clone().requires_grad_() for _ in range(2))
        ours, theirs = zoo.loss_of(case, a, y), F.cross_entropy(b.float(), y)
        assert close(ours.detach(), theirs.detach())
        ours.backward(), theirs.backward()
        assert close(a.grad, b.grad)
    if device == "cpu":
        with pytest.raises(IndexError):
            zoo.loss_of(case, out, label + 9)
