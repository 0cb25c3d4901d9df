"""GPU: what orthogonalise(out=), muon_step_ and adam_step_multi_ write counts as modified in place: a backward pass that saved the old
values raises instead of using the new ones, and a network packs its weights anew."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def S():
    import spin_nerf_amd as S
    return S


def saved(x):
    """a graph that needs x as it is now: d (w x) / d w"""
    w = torch.ones_like(x, requires_grad=True)
    return (w * x).sum()


def tensors(n, *shape):
    return [torch.randn(*shape, device="cuda", generator=torch.Generator("cuda").manual_seed(k)) for k in range(n)]


def test_what_is_written_is_modified_and_what_is_read_is_not(S):
    x, p, g, m, v = tensors(5, 6, 7)
    v = v.abs()
    calls = [(lambda: S.orthogonalise(x, out=p), (x,), (p,)), (lambda: S.orthogonalise(x, out=x), (), (x,)),
             (lambda: S.muon_step_([p], [g], [m], 0.1), (g,), (p, m)), (lambda: S.adam_step_multi_([p], [g], [m], [v], 0.1, 1), (g,), (p, m, v))]
    for call, read, written in calls:
        graphs = [(saved(t), False) for t in read] + [(saved(t), True) for t in written]
        with torch.no_grad():
            call()
        for loss, changed in graphs:
            if changed:
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    loss.backward()
            else:
                loss.backward()


def test_tensors_of_inference_mode_are_taken(S):
    with torch.inference_mode():
        x, p, g, m = tensors(4, 6, 7)
        S.orthogonalise(x, out=x)
        S.muon_step_([p], [g], [m], 0.1)
        S.adam_step_multi_([p], [g], [m], [torch.zeros_like(p)], 0.1, 1)


@pytest.mark.parametrize("how", ["muon", "adam"])
def test_a_network_packs_its_weights_anew(S, how):
    net = S.NeRF(input_ch=63, input_ch_views=27, use_viewdirs=True).cuda()
    pts, views = torch.rand(64, 3, device="cuda"), torch.nn.functional.normalize(torch.randn(64, 3, device="cuda"), dim=-1)
    flat = net.flat.detach()                         # (shares the parameter's version)
    mats, rest = net.split_hidden(flat)
    with torch.no_grad():
        before = S.mlp_query(net, pts=pts, viewdirs=views).clone()
        if how == "muon":
            S.muon_step_(mats, [torch.randn_like(t) for t in mats], [torch.zeros_like(t) for t in mats], 0.1)
        else:
            S.adam_step_multi_(rest, [torch.randn_like(t) for t in rest], [torch.zeros_like(t) for t in rest], [torch.zeros_like(t) for t in rest], 0.1, 1)
        after = S.mlp_query(net, pts=pts, viewdirs=views).clone()
        net.mark_weights_changed()
        assert torch.equal(S.mlp_query(net, pts=pts, viewdirs=views), after)
    assert not torch.equal(before, after)
