"""The zoo's heads run through the head operators and keep what they were:
the parameters' names, the numbers, and what may be done with a model."""
import json
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from k8s_device_plugin_amd.models import zoo

REPO = Path(__file__).resolve().parent.parent
GPU = pytest.param("cuda", marks=pytest.mark.gpu)


class TorchHead(nn.Module):
    """VGG-16's classifier of torch's own layers."""

    def __init__(self, c):
        super().__init__()
        self.c = nn.Sequential(
            nn.Linear(c[0].in_features, c[0].out_features), nn.ReLU(), nn.Dropout(0.5),
            nn.Linear(c[3].in_features, c[3].out_features), nn.ReLU(), nn.Dropout(0.5),
            nn.Linear(c[6].in_features, c[6].out_features))
        self.c.load_state_dict(c.state_dict())  # the same names

    def forward(self, x):
        return self.c(x)


def close(a, b):
    """Two fp32 evaluations of sums of up to 25088 terms, through 3 layers."""
    return (a.double() - b.double()).norm() <= 3 * 25088 * 2.0 ** -24 * b.double().norm()


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_vgg_classifier(device):
    torch.manual_seed(0)
    head = zoo.VGG16().classifier.eval().to(device)
    other = TorchHead(head).eval().to(device)
    x = torch.randn(2, 25088, device=device)
    y, want = head(x), other(x)
    assert close(y, want)
    g = torch.randn_like(y)
    for a, b in zip(torch.autograd.grad(y, head.parameters(), g),
                    torch.autograd.grad(want, other.parameters(), g)):
        assert close(a, b)


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_deeplab_pooled_branch(device):
    torch.manual_seed(0)
    aspp = zoo.ASPP(2048).to(device)
    assert {"gp.1.weight", "gp.2.weight", "gp.2.bias"} <= set(aspp.state_dict())
    with torch.no_grad():
        aspp.gp[2].weight.normal_()
        aspp.gp[2].bias.normal_()
    x = torch.randn(2, 2048, 5, 7, device=device)
    y, want = aspp.pooled(x), aspp.gp(x)
    assert y.shape == want.shape and close(y, want)
    used = list(aspp.gp.parameters())
    g = torch.randn_like(y)
    for a, b in zip(torch.autograd.grad(y, used, g), torch.autograd.grad(want, used, g)):
        assert close(a, b)


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_loss_is_cross_entropy(device):
    case = zoo.CASES["resnet50_train"]
    out = torch.randn(20, 1000, device=device, requires_grad=True)
    y = torch.randint(0, 1000, (20,), device=device)
    ours, theirs = zoo.loss_of(case, out, y), F.cross_entropy(out, y)
    assert close(ours.detach(), theirs.detach())
    assert close(*(torch.autograd.grad(v, out)[0] for v in (ours, theirs)))


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_distilling_one_case_from_another(device):
    dev = torch.device(device)
    case = zoo.BenchCase("student", lambda: zoo.LSTMNet(8, 16, 1, num_classes=12), "training", 4,
                         (5, 8), num_classes=12)
    student, teacher = zoo.build(case, dev), zoo.build(case, dev).eval()
    batch = zoo.distilled_batch(case, teacher, zoo.synthetic_batch(case, dev), 3)
    index, logits = batch[1]
    assert index.shape == logits.shape == (4, 3) and not logits.requires_grad
    before = [p.detach().clone() for p in student.parameters()]
    zoo.step(case, student, batch, torch.optim.SGD(student.parameters(), lr=0.1))
    assert any(not torch.equal(a, b) for a, b in zip(before, student.parameters()))
    with pytest.raises(ValueError, match="classes"):
        zoo.distilled_batch(zoo.CASES["resnet50_train"], teacher, batch, 3)
    with pytest.raises(ValueError, match="maps"):
        zoo.distilled_batch(zoo.CASES["deeplab_train"], teacher, batch, 3)


def test_command_distils(capsys, monkeypatch):
    tiny = zoo.BenchCase("tiny", lambda: zoo.LSTMNet(8, 16, 1, num_classes=12), "training", 4,
                         (5, 8), num_classes=12)
    monkeypatch.setitem(zoo.CASES, "tiny", tiny)
    zoo.main(["--cases", "tiny", "--steps", "2", "--warmup", "1", "--device", "cpu",
              "--teacher", "tiny", "--top-k", "4"])
    assert "tiny" in json.loads(capsys.readouterr().out.strip().splitlines()[-1])["samples_per_s"]


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_models_still_script_and_run_in_64_bits(device):
    head = zoo.VGG16().classifier[3].eval().to(device)
    x = torch.randn(2, 4096, device=device)
    assert close(torch.jit.script(head)(x), head(x))
    aspp = zoo.ASPP(64).double().eval().to(device)
    assert aspp(torch.randn(1, 64, 4, 4, device=device, dtype=torch.float64)).dtype == torch.float64
    fc = zoo.LSTMNet(8, 16, 1).double().to(device)
    out = fc(torch.randn(2, 3, 8, device=device, dtype=torch.float64))
    assert out.dtype == torch.float64
    zoo.loss_of(zoo.CASES["lstm_train"], out, torch.tensor([0, 1], device=device)).backward()


@pytest.mark.gpu
def test_heads_under_enforcement(tmp_path):
    """The operators' launches and memory go through the preloaded library as
    any other's: the same numbers under a quota, and an allocation beyond it
    still fails."""
    code = (
        "import json, torch\n"
        "from k8s_device_plugin_amd.models import zoo\n"
        "torch.manual_seed(0)\n"
        "head = zoo.VGG16().classifier.eval().cuda()\n"
        "x = torch.randn(3, 25088, device='cuda', requires_grad=True)\n"
        "loss = zoo.loss_of(zoo.CASES['vgg16_train'], head(x), torch.tensor([1, 2, 3], device='cuda'))\n"
        "loss.backward()\n"
        "sums = [float(p.grad.double().sum()) for p in head.parameters()] + [float(loss)]\n"
        "err = 'none'\n"
        "try: torch.empty(9 << 30, dtype=torch.uint8, device='cuda')\n"
        "except torch.cuda.OutOfMemoryError: err = 'oom'\n"
        "print(json.dumps({'sums': sums, 'err': err}))\n")
    csrc = REPO / "k8s_device_plugin_amd" / "csrc"

    def child(**env):
        out = subprocess.run([sys.executable, "-c", code], env={**os.environ, **env},
                             capture_output=True, text=True, timeout=240, cwd=REPO)
        assert out.returncode == 0, out.stderr[-2000:]
        return json.loads(out.stdout.strip().splitlines()[-1])

    free = child()
    held = child(LD_PRELOAD=str(csrc / "libvgpu-hip.so"), VGPU_DEVICE_MEMORY_LIMIT="8192m",
                 VGPU_DEVICE_MEMORY_SHARED_CACHE=str(tmp_path / "region.cache"))
    assert held["sums"] == free["sums"]
    assert (free["err"], held["err"]) == ("none", "oom")
