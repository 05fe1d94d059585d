"""Group-norm ResNets, the fused classifier loss and the Muon optimizer on the CPU primitives: against
the stock modules, the separate operators and the written-out rules; and the command line's flags."""
import os
import socket
import subprocess
import sys

import pytest
import torch

from pytorch_multiprocessing_distributed_amd.engine.optim import FusedSGD, Muon
from pytorch_multiprocessing_distributed_amd.models import build_model
from pytorch_multiprocessing_distributed_amd.ops import functional as OF
from pytorch_multiprocessing_distributed_amd.ops import torch_prims as TP
from pytorch_multiprocessing_distributed_amd.parallel.dp import DataParallel

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("name,stem", [("res", "cifar"), ("resnet50", "imagenet")])
def test_group_norm_resnet_matches_stock(name, stem):
    torch.manual_seed(0)
    f = build_model(name, num_classes=10, stem=stem, norm="group").double()
    s = build_model(name, num_classes=10, stem=stem, norm="group", impl="stock").double()
    assert list(f.state_dict()) == list(s.state_dict())
    s.load_state_dict(f.state_dict())
    x, y = torch.randn(3, 3, 32, 32, dtype=torch.float64), torch.randint(0, 10, (3,))
    lf = OF.cross_entropy(f(x.permute(0, 2, 3, 1).contiguous()), y)
    ls = torch.nn.functional.cross_entropy(s(x), y)
    lf.backward()
    ls.backward()
    # one network in fp64 with its sums in another order; two dozen (fifty) normalised layers multiply
    # roundings of 2^-53 by far less than 1e5
    assert abs(lf.item() - ls.item()) < 1e-11
    for (n, p), q in zip(f.named_parameters(), s.parameters()):
        # the classifier's own gradients are kept in fp32 by ops.functional.linear: each entry is rounded by
        # up to 2^-24 of itself, so the matrix by up to 2^-24 of its norm
        own = 2.0 ** -24 if n.startswith("linear.") else 0.0
        assert (p.grad - q.grad).norm() <= (1e-10 + own) * q.grad.norm() + 1e-12, n


def test_fused_loss_is_the_separate_loss():
    torch.manual_seed(1)
    m = build_model("res", norm="group").double()
    x, y = torch.randn(4, 16, 16, 3, dtype=torch.float64), torch.randint(0, 10, (4,))
    loss, correct = m(x, y)
    out = m(x)
    ref = OF.cross_entropy(out, y)
    names, params = zip(*m.named_parameters())
    ga, gb = torch.autograd.grad(loss, params), torch.autograd.grad(ref, params)
    assert abs(loss.item() - ref.item()) < 1e-13 and correct.item() == OF.correct_count(out, y).item()
    for n, a, b in zip(names, ga, gb):
        # the separate classifier's gradients are rounded to fp32 (2^-24 of each entry)
        own = 2.0 ** -24 if n.startswith("linear.") else 0.0
        assert (a - b).norm() <= (1e-11 + own) * b.norm(), n
    with pytest.raises(ValueError, match="logits only"):
        build_model("res", impl="stock")(x.permute(0, 3, 1, 2), y)


def test_model_refusals():
    with pytest.raises(ValueError, match="norm"):
        build_model("res", norm="layer")


def _small():
    torch.manual_seed(2)
    return build_model("res")


def _fill_grads(m, seed):
    g = torch.Generator().manual_seed(seed)
    for _, p in sorted(m.named_parameters()):
        p.grad.copy_(torch.randn(p.shape, generator=g))


@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_rule(nesterov):
    m = _small()
    ref = {n: p.detach().double().clone() for n, p in m.named_parameters()}
    buf = {}
    opt = Muon(m, lr=0.03, momentum=0.9, weight_decay=0.01, nesterov=nesterov, rest_lr=0.2, rest_momentum=0.8,
               rest_weight_decay=1e-3)
    for step in range(3):
        _fill_grads(m, step)
        for n, p in m.named_parameters():
            g = p.grad.double()
            mat = p.dim() == 4
            mom = 0.9 if mat else 0.8
            if not mat:
                g = g + 1e-3 * ref[n]
            buf[n] = g.clone() if step == 0 else mom * buf[n] + g
            u = g + mom * buf[n] if (nesterov or not mat) else buf[n]
            if mat:
                d = torch.empty(p.shape[0], p.numel() // p.shape[0], dtype=torch.float64)
                TP.newton_schulz_([u.flatten(1)], [d], 5, OF.NS_COEFFS, 1e-7, [1.0])
                scale = max(1.0, d.shape[0] / d.shape[1]) ** 0.5
                ref[n] = ref[n] * (1 - 0.03 * 0.01) - 0.03 * scale * d.reshape(p.shape)
            else:
                ref[n] = ref[n] - 0.2 * u
        opt.step()
    # fp32 against fp64: orthogonalised entries are a hundred roundings off and up to 1.3 (rates 0.03 and
    # below 0.1 with the factor), the others a few roundings of values below 10
    for n, p in m.named_parameters():
        assert (p.double() - ref[n]).abs().max() <= 3 * 0.1 * 1.3 * 485 * 100 * 2.0 ** -24 + 1e-5, n
        assert (p.double() - ref[n]).norm() <= 1e-5 * ref[n].norm() + 1e-5, n


def test_muon_follows_the_arena_and_resumes():
    a, b = _small(), _small()
    oa, ob = Muon(a), Muon(b)
    _fill_grads(a, 0)
    _fill_grads(b, 0)
    oa.step()
    ob.step()
    oa.flat.relayout(list(reversed(range(len(oa.flat.params)))))
    sd = ob.state_dict()
    c = _small()
    c.load_state_dict(b.state_dict())
    oc = Muon(c)
    oc.load_state_dict(sd)
    for m, o in ((a, oa), (b, ob), (c, oc)):
        _fill_grads(m, 1)
        o.step()
    for p, q, r in zip(a.parameters(), b.parameters(), c.parameters()):
        assert torch.equal(p, q) and torch.equal(q, r)


def test_muon_groups_schedule_and_refusals():
    m = _small()
    opt = Muon(m, lr=0.02, rest_lr=0.1)
    sch = torch.optim.lr_scheduler.MultiStepLR(opt, [1], gamma=0.5)
    opt.step()
    sch.step()
    assert [g["lr"] for g in opt.param_groups] == [0.01, 0.05]
    assert all(p.dim() == 4 for p in opt.param_groups[0]["params"])
    with pytest.raises(ValueError, match="Nesterov"):
        Muon(_small(), momentum=0.0)
    with pytest.raises(ValueError, match="step"):
        Muon(_small(), ns_steps=0)
    m = _small()
    with pytest.raises(ValueError, match="two dimensions"):
        Muon(m, matrices=[m.bn1.weight])
    with pytest.raises(ValueError, match="not a trainable"):
        Muon(_small(), matrices=[torch.nn.Parameter(torch.zeros(2, 2))])
    m = _small()
    only = Muon(m, matrices=[m.linear.weight])
    assert len(only.param_groups[0]["params"]) == 1
    _fill_grads(m, 0)
    only.step()


def test_muon_refuses_matrices_past_its_sides():
    from pytorch_multiprocessing_distributed_amd.engine.optim import Muon
    lin = torch.nn.Linear(2, 2 ** 20 + 1, bias=False)
    with pytest.raises(ValueError, match="at most 2\\^20"):
        Muon(lin, matrices=[lin.weight])


def test_muon_without_matrices_is_sgd():
    a, b = _small(), _small()
    oa = Muon(a, matrices=[], rest_lr=0.1, rest_momentum=0.9, rest_weight_decay=1e-4)
    ob = FusedSGD(b, lr=0.1, momentum=0.9, weight_decay=1e-4, nesterov=True)
    for k in range(3):
        _fill_grads(a, k)
        _fill_grads(b, k)
        oa.step()
        ob.step()
    for p, q in zip(a.parameters(), b.parameters()):
        # the same rule in another order of fp32 operations
        assert (p - q).abs().max() <= 32 * 2.0 ** -24 * 10


def test_a_step_of_all_three():
    torch.manual_seed(3)
    m = DataParallel(build_model("res", norm="group"), None)
    opt = Muon(m)
    x, y = torch.randn(4, 16, 16, 3), torch.randint(0, 10, (4,))
    for _ in range(2):
        loss, _ = m(x, y)
        opt.zero_grad()
        loss.backward()
        opt.step()
    assert loss.isfinite() and all(p.isfinite().all() for p in m.parameters())


def _free_port():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    p = s.getsockname()[1]
    s.close()
    return p


@pytest.mark.slow
def test_main_py_with_the_flags(tmp_path):
    save = str(tmp_path / "run")
    cmd = [sys.executable, os.path.join(ROOT, "main.py"), "--world_size", "2", "--backend", "gloo", "--device", "cpu",
           "--synthetic", "--epochs", "1", "--max_steps", "2", "--eval_batches", "1", "--batch_size", "8",
           "--train_samples", "64", "--save_path", save, "--print-freq", "1", "--no_plot",
           "--norm", "group", "--loss", "fused", "--optimizer", "muon",
           "--master_port", str(_free_port())]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=300, cwd=ROOT,
                       env=dict(os.environ, MASTER_ADDR="127.0.0.1"))
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-3000:]
    assert "Epoch: [1][1/" in r.stdout and "Accuracy" in r.stdout, r.stdout[-2000:]
    sd = torch.load(os.path.join(save, "model_1.pth"), map_location="cpu", weights_only=True)
    assert "module.bn1.weight" in sd and not any("running" in k for k in sd)
