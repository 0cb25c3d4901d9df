"""GPU: RenderTrainer(muon=...) — the training step with orthogonalised updates, eagerly and as a captured graph."""
import importlib

import pytest
import torch

from test_gpu_train_step import _two_trainers
from test_gpu_muon import bound32, muon_oracle

pytestmark = pytest.mark.gpu


def trainers(graph=False, muon=True, precision="bf16"):
    train = importlib.import_module("spin-nerf_amd.train")
    (a, b), hwf, rays, target, _ = _two_trainers(precision, 128)
    ta = train.RenderTrainer(a[0].kw, lrate=5e-4, muon=muon)
    tb = train.RenderTrainer(b[0].kw, lrate=5e-4, graph=graph, muon=muon)
    return ta, tb, hwf, rays, target


def test_a_step_is_the_formula_on_its_gradients():
    ta, _, hwf, rays, target = trainers(muon=dict(weight_decay=0.1))
    ta.step(*hwf, rays, target)
    before = [(n.flat.detach().clone(), m.clone(), v.clone()) for n, m, v in zip(ta.nets, ta.m, ta.v)]
    ta.step(*hwf, rays, target)
    for (p0, m0, v0), n, m, v in zip(before, ta.nets, ta.m, ta.v):
        hidden = n.hidden_matrices()
        view = n.named_views
        for k in view():
            P, G, M, V = (view(t)[k] for t in (p0, n.flat.grad, m0, v0))
            got, gm, gv = view(n.flat.detach())[k], view(m)[k], view(v)[k]
            if k in hidden:
                rp, rm, step, o, norms = muon_oracle(P, G, M, 5e-4, 0.95, True, 0.1, "rms", 1.0)
                assert float((gm.cpu().double() - rm).norm()) <= 3 * 2.0 ** -24 * float(rm.norm() + G.double().norm())
                tol = step * (bound32(norms, 5, 3.4445) + 485 * 4 * 2.0 ** -24) + 4 * 2.0 ** -24 * P.double().norm().cpu()
                assert float((got.cpu().double() - rp).norm()) <= float(tol), k
                assert not bool(gv.any())
            else:
                G, M, V = G.double(), M.double(), V.double()
                M, V = 0.9 * M + 0.1 * G, 0.999 * V + 0.001 * G * G
                ref = P.double() - 5e-4 * (M / (1 - 0.9 ** 2)) / ((V / (1 - 0.999 ** 2)).sqrt() + 1e-8)
                # 1 - beta2 in 32 bits is off by 1.3e-5 of itself; a step is a few times the rate at most
                assert float((got.double() - ref).abs().max()) <= 10 * 5e-4 * 2e-5 + 4 * 2.0 ** -24 * float(P.abs().max()), k


def test_graph_replayed_step_equals_the_eager_step():
    ta, tb, hwf, rays, target = trainers(graph=True)
    g = torch.Generator().manual_seed(11)
    batches = [(rays[:, s].contiguous(), target[s].contiguous()) for s in (torch.randperm(rays.shape[1], generator=g).cuda() for _ in range(6))]
    la = [float(ta.step(*hwf, r, t)[0]) for r, t in batches]
    lb = []
    for k, (r, t) in enumerate(batches):
        lb.append(float(tb.step(*hwf, r, t)[0]))
        torch.randn(1000, device="cuda").sum().item()          # other eager work between replays
    assert tb._graph is not None, "the graph route was not taken"
    assert all(abs(x - y) <= 1e-5 * abs(x) for x, y in zip(la, lb)), (la, lb)
    for na, nb in zip(ta.nets, tb.nets):
        assert float((na.flat.detach() - nb.flat.detach()).abs().max()) <= 2e-6
    # (moments and momentum of the two routes: the same kernels on the same gradients)
    for x, y in zip(ta.m + ta.v, tb.m + tb.v):
        assert float((x - y).abs().max()) <= 1e-6 * float(x.abs().max()) + 1e-12


def test_a_step_leaves_the_other_route_and_adam_as_they_were():
    """Adam without muon: the same bits as ever, whatever ran before it"""
    train = importlib.import_module("spin-nerf_amd.train")
    (a, b), hwf, rays, target, _ = _two_trainers("bf16", 128)
    la = float(a[0].step(*hwf, rays, target)[0])
    c = train.RenderTrainer(b[0].kw, lrate=5e-4)
    lb = float(c.step(*hwf, rays, target)[0])
    assert abs(la - lb) <= 1e-5 * abs(la)          # (the loss is a sum of atomics: its order moves the last bits)
    for na, nb in zip(a[0].nets, c.nets):
        assert torch.equal(na.flat.detach(), nb.flat.detach())


def test_checkpoint_resumes_on_the_device(tmp_path):
    ta, tb, hwf, rays, target = trainers(muon=dict(precision="fp16"))
    for _ in range(2):
        ta.step(*hwf, rays, target)
    path = str(tmp_path / "000002.tar")
    ta.save_checkpoint(path)
    tb.load_checkpoint(path)
    tb._draws = ta._draws
    tb._seed = ta._seed
    la, lb = float(ta.step(*hwf, rays, target)[0]), float(tb.step(*hwf, rays, target)[0])
    assert abs(la - lb) <= 1e-5 * abs(la)          # (the loss is a sum of atomics: its order moves the last bits)
    for na, nb in zip(ta.nets, tb.nets):
        assert torch.equal(na.flat.detach(), nb.flat.detach())
