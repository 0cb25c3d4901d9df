"""CPU: a run trained with RenderTrainer(muon=...) resumes through create_nerf, and only as such a run; the kernels are replaced by the
formulas in torch, as in test_muon_trainer_cpu.py."""
import argparse

import pytest
import torch

from test_muon_trainer_cpu import set_grads, train  # noqa: F401  (a fixture)

CPU = torch.device("cpu")


@pytest.fixture
def args(tmp_path):
    (tmp_path / "run").mkdir()
    return argparse.Namespace(multires=10, multires_views=4, i_embed=0, use_viewdirs=True, N_importance=128, N_samples=64,
                              alpha_model_path=None, netdepth=8, netwidth=256, netdepth_fine=8, netwidth_fine=256, netchunk=65536,
                              lrate=1e-3, basedir=str(tmp_path), expname="run", ft_path=None, no_reload=False, perturb=1.0,
                              white_bkgd=True, raw_noise_std=1.0, dataset_type="llff", no_ndc=True, lindisp=True, sigma_loss=False,
                              no_coarse=False)


def steps(tr, seeds):
    for k in seeds:
        set_grads(tr.nets, k)
        tr.apply_gradients()


def trained(train, args, path, **kw):  # noqa: F811
    import spin_nerf_amd as S
    torch.manual_seed(3)
    kws, _, start, _, opt = S.create_nerf(args, device=CPU)
    tr = train.RenderTrainer(kws, lrate=1e-3, lrate_decay=1, optimizer=opt, start=start, **kw)
    steps(tr, range(3))
    tr.save_checkpoint(str(path))
    return tr


def test_resume_through_create_nerf_continues_like_an_uninterrupted_run(train, args, tmp_path):  # noqa: F811
    import spin_nerf_amd as S
    muon = dict(weight_decay=0.1)
    tr = trained(train, args, tmp_path / "run" / "000003.tar", muon=muon)
    steps(tr, (7, 8))                                               # the uninterrupted run
    kws, _, start, _, opt = S.create_nerf(args, device=CPU)         # picks the checkpoint up
    assert start == 3
    tr2 = train.RenderTrainer(kws, lrate=1e-3, lrate_decay=1, optimizer=opt, start=start, muon=muon)
    assert tr2.opt_step == 3 and tr2.global_step == 3 and abs(tr2.current_lr() - 1e-3 * 0.1 ** (2 / 1000)) < 1e-12
    steps(tr2, (7, 8))
    for a, b in zip(tr.nets, tr2.nets):
        assert torch.equal(a.flat.detach(), b.flat.detach())
    for a, b in zip(tr.m + tr.v, tr2.m + tr2.v):
        assert torch.equal(a, b)


def test_its_weights_load_for_rendering(train, args, tmp_path):  # noqa: F811
    import spin_nerf_amd as S
    tr = trained(train, args, tmp_path / "elsewhere.tar", muon=True)
    args.ft_path = str(tmp_path / "elsewhere.tar")
    _, kw_test, start, _, _ = S.create_nerf(args, device=CPU)
    assert start == 3
    for n, k in zip(tr.nets, ("network_fn", "network_fine")):
        assert torch.equal(n.flat.detach(), kw_test[k].flat.detach())


def test_adam_does_not_take_momentum_buffers_nor_muon_adams_moments(train, args, tmp_path, monkeypatch):  # noqa: F811
    import spin_nerf_amd as S
    from test_checkpoint_cpu import _cpu_adam
    monkeypatch.setattr(train.ops, "adam_step_", _cpu_adam)
    trained(train, args, tmp_path / "run" / "000003.tar", muon=True)
    kws, _, start, _, opt = S.create_nerf(args, device=CPU)
    with pytest.raises(RuntimeError, match="momentum buffer"):
        train.RenderTrainer(kws, optimizer=opt, start=start)
    for n in (kws["network_fn"], kws["network_fine"]):
        n.flat.grad = torch.ones_like(n.flat)
    with pytest.raises(KeyError, match="exp_avg"):                  # torch's own Adam: no silent restart of its moments either
        opt.step()
    args.no_reload = True
    trained(train, args, tmp_path / "run" / "000004.tar")
    args.no_reload = False
    kws, _, start, _, opt = S.create_nerf(args, device=CPU)
    with pytest.raises(RuntimeError, match="Adam state"):
        train.RenderTrainer(kws, optimizer=opt, start=start, muon=True)


def test_a_state_that_does_not_fit_is_refused(train, args, tmp_path):  # noqa: F811
    import spin_nerf_amd as S
    path = tmp_path / "run" / "000003.tar"
    trained(train, args, path, muon=True)
    whole = torch.load(path, weights_only=True)
    for spoil, why in ((lambda st: st.pop(5), "no Adam state"),
                       (lambda st: st.__setitem__(2, dict(st[2], momentum_buffer=st[2]["momentum_buffer"][1:])), "elements"),
                       (lambda st: st.__setitem__(2, dict(step=st[2]["step"], exp_avg=torch.zeros(256, 256), exp_avg_sq=torch.zeros(256, 256))), "Adam moments")):
        ck = dict(whole, optimizer_state_dict=dict(whole["optimizer_state_dict"], state=dict(whole["optimizer_state_dict"]["state"])))
        spoil(ck["optimizer_state_dict"]["state"])
        torch.save(ck, path)
        with pytest.raises(RuntimeError, match=why):
            S.create_nerf(args, device=CPU)


@pytest.mark.parametrize("muon", [True, None])
def test_a_refused_checkpoint_leaves_the_trainer_as_it_was(train, args, tmp_path, monkeypatch, muon):  # noqa: F811
    from test_checkpoint_cpu import _cpu_adam
    monkeypatch.setattr(train.ops, "adam_step_", _cpu_adam)
    args.no_reload = True
    other = tmp_path / "other.tar"
    trained(train, args, other, muon=None if muon else True)          # the other kind's
    tr = trained(train, args, tmp_path / "own.tar", muon=muon)
    steps(tr, (5,))
    now = lambda: [t.detach().clone() for t in [n.flat for n in tr.nets] + tr.m + tr.v]  # noqa: E731
    before, counts = now(), (tr.opt_step, tr.global_step, tr.current_lr())
    with pytest.raises(RuntimeError, match="momentum buffer"):
        tr.load_checkpoint(str(other))
    assert all(torch.equal(a, b) for a, b in zip(before, now())) and counts == (tr.opt_step, tr.global_step, tr.current_lr())
    tr.load_checkpoint(str(tmp_path / "own.tar"))                     # and its own loads as ever
    assert tr.opt_step == 3 and not torch.equal(before[0], tr.nets[0].flat.detach())
