"""CPU: RenderTrainer(muon=...) — which parameters go where, checkpoints, refusals, and two ranks over gloo.  The kernels are replaced by
the formulas in torch; their own tests are tests/test_gpu_muon.py."""
import importlib
import os
import sys

import pytest
import torch
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def cpu_orth(x, steps, coefficients, eps):
    a, b, c = coefficients
    X = x.double()
    X = X / X.norm().clamp(min=eps)
    for _ in range(steps):
        A = X @ X.T
        X = a * X + (b * A + c * A @ A) @ X
    return X


def cpu_muon(params, grads, bufs, lr, momentum, nesterov, weight_decay, scale, steps, coefficients, eps, grad_scale, precision, state=None):
    for p, g, m in zip(params, grads, bufs):
        g = g * grad_scale
        m.mul_(momentum).add_(g)
        o = cpu_orth(g + momentum * m if nesterov else m, steps, coefficients, eps)
        q = {"rms": 0.2 * max(p.shape) ** 0.5, "spectral": max(1.0, p.shape[0] / p.shape[1]) ** 0.5, "none": 1.0}[scale]
        p.copy_(p.double() * (1 - lr * weight_decay) - lr * q * o)


def cpu_adam_multi(params, grads, ms, vs, lr, step, beta1=0.9, beta2=0.999, eps=1e-8, grad_scale=1.0, state=None):
    for p, g, m, v in zip(params, grads, ms, vs):
        g = g * grad_scale
        m.mul_(beta1).add_(g, alpha=1 - beta1)
        v.mul_(beta2).addcmul_(g, g, value=1 - beta2)
        p.addcdiv_(m / (1 - beta1 ** step), (v / (1 - beta2 ** step)).sqrt() + eps, value=-lr)


@pytest.fixture
def train(monkeypatch):
    t = importlib.import_module("spin-nerf_amd.train")
    monkeypatch.setattr(t.ops, "muon_step_", cpu_muon)
    monkeypatch.setattr(t.ops, "adam_step_multi_", cpu_adam_multi)
    return t


def nets(n=2, seed=0):
    import spin_nerf_amd as S
    torch.manual_seed(seed)
    return [S.NeRF(input_ch=63, input_ch_views=27, use_viewdirs=True) for _ in range(n)]


def set_grads(ns, seed):
    g = torch.Generator().manual_seed(seed)
    for n in ns:
        n.flat.grad = torch.randn(n.flat.shape, generator=g) * 1e-2


def test_hidden_matrices_and_the_rest_cover_the_parameters():
    import spin_nerf_amd as S
    for vd, och, n_mats in ((True, 4, 9), (False, 5, 7)):
        n = S.NeRF(input_ch=63, input_ch_views=27 if vd else 0, output_ch=och, use_viewdirs=vd)
        mark = torch.zeros_like(n.flat.data)
        mats, rest = n.split_hidden(mark)
        assert len(mats) == n_mats and all(m.dim() == 2 and min(m.shape) >= 128 for m in mats) and all(r.dim() == 1 for r in rest)
        for t in mats + rest:
            assert t.untyped_storage().data_ptr() == mark.untyped_storage().data_ptr()
            t += 1
        assert bool((mark == 1).all())
    rgb = S.NeRF_RGB(input_ch=63, input_ch_views=27, use_viewdirs=True)
    assert len(rgb.split_hidden()[0]) == 9


def test_step_moves_hidden_matrices_by_the_orthogonalised_update(train):
    ns = nets()
    before = [n.flat.detach().clone() for n in ns]
    tr = train.RenderTrainer({"network_fn": ns[0], "network_fine": ns[1]}, lrate=1e-3, muon=True)
    set_grads(ns, 1)
    tr.apply_gradients()
    for n, b in zip(ns, before):
        hidden = n.hidden_matrices()
        for (k, p), o, g in zip(n.named_views(n.flat.detach()).items(), n.named_views(b).values(), n.named_views(n.flat.grad).values()):
            d = (p - o).double() / 1e-3
            if k in hidden:        # singular values near one; but five steps lift the least ones by 3.4445 ** 5 = 485 only, and a random
                                   # 256 x 256 matrix has some at 1 / 16 where its norm is 256
                s = torch.linalg.svdvals(d / (0.2 * max(d.shape) ** 0.5))
                assert float(s.median()) > 0.6 and float(s.max()) < 1.3, (k, float(s.median()), float(s.max()))
            else:                  # Adam's first step: the gradient's sign, but for eps
                assert float((d + g / (g.abs() + 1e-8)).abs().max()) < 1e-3, k


def test_a_network_without_a_gradient_takes_no_step(train):
    ns = nets()
    tr = train.RenderTrainer({"network_fn": ns[0], "network_fine": ns[1]}, lrate=1e-3, muon=True)
    set_grads(ns, 2)
    ns[1].flat.grad = None
    before = ns[1].flat.detach().clone()
    tr.apply_gradients()
    assert torch.equal(ns[1].flat.detach(), before) and float(tr.m[1].abs().max()) == 0


def test_checkpoint_round_trip_and_what_it_refuses(train, tmp_path):
    ns = nets()
    tr = train.RenderTrainer({"network_fn": ns[0], "network_fine": ns[1]}, lrate=1e-3, muon=dict(weight_decay=0.1))
    for k in range(3):
        set_grads(ns, k); tr.apply_gradients()
    path = str(tmp_path / "000003.tar")
    tr.save_checkpoint(path)
    ns2 = nets(seed=5)
    tr2 = train.RenderTrainer({"network_fn": ns2[0], "network_fine": ns2[1]}, lrate=1e-3, muon=dict(weight_decay=0.1))
    tr2.load_checkpoint(path)
    assert tr2.global_step == 3 and tr2.opt_step == 3 and tr2.current_lr() == tr.current_lr()
    for k in (7, 8):
        set_grads(ns, k); tr.apply_gradients()
        set_grads(ns2, k); tr2.apply_gradients()
    for a, b in zip(ns, ns2):
        assert torch.equal(a.flat, b.flat)
    # Adam does not resume from momentum buffers, nor muon from Adam's moments
    ns3 = nets()
    plain = train.RenderTrainer({"network_fn": ns3[0], "network_fine": ns3[1]})
    with pytest.raises(RuntimeError, match="momentum buffer"):
        plain.load_checkpoint(path)
    plain = train.RenderTrainer({"network_fn": ns3[0], "network_fine": ns3[1]})
    plain.opt_step = 1
    plain.save_checkpoint(str(tmp_path / "adam.tar"))
    with pytest.raises(RuntimeError, match="Adam moments"):
        tr2.load_checkpoint(str(tmp_path / "adam.tar"))


def test_settings_and_networks_that_are_refused(train):
    import spin_nerf_amd as S
    ns = nets(1)
    with pytest.raises(ValueError, match="no settings"):
        train.RenderTrainer({"network_fn": ns[0]}, muon=dict(momentun=0.9))
    with pytest.raises(NotImplementedError, match="NeRF_TCNN"):
        train.RenderTrainer({"network_fn": S.NeRF_TCNN()}, muon=True)
    opt = torch.optim.Adam([ns[0].flat], lr=1e-3)
    opt.state[ns[0].flat] = {"step": torch.tensor(2.0), "exp_avg": torch.zeros_like(ns[0].flat), "exp_avg_sq": torch.zeros_like(ns[0].flat)}
    with pytest.raises(RuntimeError, match="Adam state"):
        train.RenderTrainer({"network_fn": ns[0]}, optimizer=opt, start=2, muon=True)
    train.RenderTrainer({"network_fn": ns[0]}, optimizer=torch.optim.Adam([ns[0].flat], lr=1e-3), start=0, muon=True)


def _worker(rank, world, port, out):
    sys.path.insert(0, ROOT)
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    import torch.distributed as dist
    torch.set_num_threads(2)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    t = importlib.import_module("spin-nerf_amd.train")
    t.ops.muon_step_, t.ops.adam_step_multi_ = cpu_muon, cpu_adam_multi
    ns = nets(2, seed=rank)
    tr = t.RenderTrainer({"network_fn": ns[0], "network_fine": ns[1]}, lrate=1e-3, world_size=world, muon=True)
    tr.broadcast_parameters()
    start = [n.flat.detach().clone() for n in ns]
    for k in range(2):
        set_grads(ns, 10 * k + rank)
        tr.apply_gradients()
    torch.save({"start": start, "end": [n.flat.detach() for n in ns]}, f"{out}.{rank}")
    dist.destroy_process_group()


def test_two_ranks_step_alike_on_the_mean_gradient(train, tmp_path):
    import socket
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    out = str(tmp_path / "r")
    mp.spawn(_worker, args=(2, port, out), nprocs=2, join=True)
    a, b = torch.load(out + ".0", weights_only=True), torch.load(out + ".1", weights_only=True)
    ns = nets()
    for n, x, y in zip(ns, a["start"], b["start"]):
        assert torch.equal(x, y)
        n.flat.data.copy_(x)
    for x, y in zip(a["end"], b["end"]):
        assert torch.equal(x, y)
    tr = train.RenderTrainer({"network_fn": ns[0], "network_fine": ns[1]}, lrate=1e-3, muon=True)
    for k in range(2):
        set_grads(ns, 10 * k)
        g0 = [n.flat.grad.clone() for n in ns]
        set_grads(ns, 10 * k + 1)
        for n, g in zip(ns, g0):
            n.flat.grad = (n.flat.grad + g) * 0.5
        tr.apply_gradients()
    for n, x in zip(ns, a["end"]):
        assert float((n.flat.detach() - x).abs().max()) < 1e-6
