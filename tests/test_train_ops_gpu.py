"""Group-norm ResNet, fused classifier loss and Muon together on the gfx950 kernels: gradients of a whole
model, the optimizer's step, the captured step, the program's command line."""
import copy
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _rel(a, b):
    a, b = a.double(), b.double()
    return ((a - b).norm() / b.norm().clamp_min(1e-30)).item()


def _grads(m0, x, y, torch_prims, fused):
    from pytorch_multiprocessing_distributed_amd.engine.train import loss_of
    from pytorch_multiprocessing_distributed_amd.ops import functional as OF
    m = copy.deepcopy(m0)
    OF.force_torch_prims(torch_prims)
    try:
        loss, _, _ = loss_of(m, x, y, fused)
        loss.backward()
    finally:
        OF.force_torch_prims(False)
    torch.cuda.synchronize()
    return loss.item(), {n: p.grad for n, p in m.named_parameters()}


@pytest.mark.parametrize("name,stem,size,batch", [("res", "cifar", 32, 64), ("resnet50", "imagenet", 96, 8)])
def test_model_gradients(name, stem, size, batch):
    """One step of the whole model on the kernels against the reference primitives in fp32, with the
    reference primitives on bf16 activations as the yardstick of what those cost: every tensor within
    three times its error (or half the median's, where it happens to be small) plus one bf16 step."""
    from pytorch_multiprocessing_distributed_amd.models import build_model
    from pytorch_multiprocessing_distributed_amd.ops.native import C
    torch.manual_seed(0)
    m0 = build_model(name, num_classes=100, stem=stem, norm="group").cuda()
    x, y = C.synth_images(batch, size, size, 8, 3, 100, 7, 0)
    lf, f32 = _grads(m0, x.float(), y, True, False)
    lb, ref = _grads(m0, x, y, True, False)
    for fused in (False, True):
        lh, hip = _grads(m0, x, y, False, fused)
        assert abs(lh - lf) <= 3 * abs(lb - lf) + 2.0 ** -7 * lf
        eh = {n: _rel(hip[n], f32[n]) for n in f32}
        eb = {n: _rel(ref[n], f32[n]) for n in f32}
        floor = 0.5 * sorted(eb.values())[len(eb) // 2]
        bad = [(n, eh[n], eb[n]) for n in eh if eh[n] > 3.0 * max(eb[n], floor) + 2.0 ** -7]
        assert not bad, bad[:8]


def test_muon_step_matches_the_primitives():
    from pytorch_multiprocessing_distributed_amd.engine.optim import Muon
    from pytorch_multiprocessing_distributed_amd.models import build_model
    torch.manual_seed(1)
    m0 = build_model("res", norm="group")
    a, b = copy.deepcopy(m0).cuda(), copy.deepcopy(m0)
    kw = dict(lr=0.02, weight_decay=0.01)
    oa, ob = Muon(a, **kw), Muon(b, **kw)
    for k in range(3):
        g = torch.Generator().manual_seed(k)
        for p, q in zip(a.parameters(), b.parameters()):
            r = torch.randn(q.shape, generator=g)
            p.grad.copy_(r)
            q.grad.copy_(r)
        oa.step()
        ob.step()
    for (n, p), q in zip(a.named_parameters(), b.named_parameters()):
        q = q[1]
        # each side's direction is 50 roundings of 2^-22 (its matrix's norm) from the exact one
        # (test_newton_schulz_gpu.py), three steps of it at rate 0.02 and a factor of at most 2
        d = 3 * 0.02 * 2 * min(p.shape[0], p.numel() // p.shape[0]) ** 0.5 * 1.2 if p.dim() == 4 else 0.0
        assert (p.cpu() - q).double().norm() <= 2 * 100 * 2.0 ** -22 * d + 32 * 2.0 ** -24 * (q.double().norm() + 10), n


def _steps(graph, m0, batches):
    from pytorch_multiprocessing_distributed_amd.engine.optim import Muon
    from pytorch_multiprocessing_distributed_amd.engine.train import GraphedStep, loss_of
    from pytorch_multiprocessing_distributed_amd.ops import functional as OF
    from pytorch_multiprocessing_distributed_amd.parallel.dp import DataParallel
    m = DataParallel(copy.deepcopy(m0), None)
    opt = Muon(m, lr=0.01)
    g, rows = None, []
    for i, (x, y) in enumerate(batches):
        if i == 4:
            for grp in opt.param_groups:
                grp["lr"] *= 0.5                     # a scheduler step between replays
        if graph and i == 2:
            g = GraphedStep(m, opt, x, y, True)
        if g is not None:
            _, loss = g(x, y)
            correct = g.correct
        else:
            loss, correct, _ = loss_of(m, x, y, True)
            opt.zero_grad()
            loss.backward(OF.loss_seed(loss))
            opt.step()
        rows.append(torch.stack([loss.detach().double(), correct[0].double()]))
        with torch.no_grad():
            loss_of(m, x, y, True)                   # the program's own eager work between replays
        torch.cuda.synchronize()
    assert opt.steps == len(batches)
    return torch.stack(rows), opt.flat.param_arena.clone(), opt.momentum_arena.clone()


def test_muon_refuses_before_any_step():
    from pytorch_multiprocessing_distributed_amd.engine.optim import Muon
    for kw, match in ((dict(ns_coeffs=(50.0, 0.0, 0.0)), "range"), (dict(ns_steps=65), "steps"),
                      (dict(eps=-1.0), "eps")):
        with pytest.raises(RuntimeError, match=match):
            Muon(torch.nn.Conv2d(8, 8, 3).cuda(), **kw)


def test_captured_step_is_bit_exact():
    from pytorch_multiprocessing_distributed_amd.models import build_model
    from pytorch_multiprocessing_distributed_amd.ops import functional as OF
    from pytorch_multiprocessing_distributed_amd.ops.native import C
    OF.set_wgrad_stream(False)
    try:
        torch.manual_seed(0)
        m0 = build_model("res", num_classes=10, norm="group").cuda()
        batches = [C.synth_images(32, 32, 32, 8, 3, 10, 7 + s, 0) for s in range(6)]
        st = torch.cuda.Stream()                     # captures need another stream than the default one
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            _steps(False, m0, batches)               # tunes the convolutions' kernel choices
            eager, again, graph = _steps(False, m0, batches), _steps(False, m0, batches), _steps(True, m0, batches)
    finally:
        OF.set_wgrad_stream(True)
    for a, b, g in zip(eager, again, graph):
        assert torch.equal(a, b) and torch.equal(a, g)


@pytest.mark.slow
def test_main_py_with_the_flags_on_gpu(tmp_path):
    save = str(tmp_path / "run")
    cmd = [sys.executable, os.path.join(ROOT, "main.py"), "--world_size", "1", "--synthetic", "--epochs", "1",
           "--max_steps", "6", "--eval_batches", "2", "--batch_size", "32", "--train_samples", "512",
           "--save_path", save, "--print-freq", "2", "--no_plot", "--norm", "group", "--loss", "fused",
           "--optimizer", "muon", "--master_port", "29741"]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=100, cwd=ROOT,
                       env=dict(os.environ, MASTER_ADDR="127.0.0.1"))
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-3000:]
    assert "step mode: graph" in r.stdout and "Epoch: [1][4/" in r.stdout and "Accuracy" in r.stdout, r.stdout[-2000:]
