"""CPU: what RenderTrainer(muon=...) takes as settings, and that it refuses the others when it is made."""
import pytest
import torch

from test_muon_trainer_cpu import nets, set_grads, train  # noqa: F401  (a fixture)


def test_an_empty_dict_asks_for_the_defaults(train):  # noqa: F811
    a = train.RenderTrainer({"network_fn": nets(1)[0]}, lrate=1e-3, muon={})
    b = train.RenderTrainer({"network_fn": nets(1)[0]}, lrate=1e-3, muon=True)
    assert a.muon is not None and a.muon == b.muon
    for t in (a, b):
        set_grads(t.nets, 1)
        t.apply_gradients()
    assert torch.equal(a.nets[0].flat, b.nets[0].flat)
    for off in (None, False, 0):
        assert train.RenderTrainer({"network_fn": nets(1)[0]}, muon=off).muon is None


@pytest.mark.parametrize("bad", ["spectral", 2, 0.95, [], ("momentum", 0.9), torch.tensor(True)])
def test_neither_a_dict_nor_a_truth_value_is_refused(train, bad):  # noqa: F811
    with pytest.raises(ValueError, match="True or a dict"):
        train.RenderTrainer({"network_fn": nets(1)[0]}, muon=bad)


@pytest.mark.parametrize("bad,why", [(dict(precision="bf16"), "precision"), (dict(precision=None), "precision"), (dict(scale="adam"), "scale"),
                                     (dict(steps=0), "steps"), (dict(steps=2.5), "steps"), (dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"),
                                     (dict(coefficients=(16.0, 0.0, 0.0)), "singular values"), (dict(coefficients=(3.0, -4.0)), "three"),
                                     (dict(coefficients=(float("nan"), 0.0, 0.0)), "singular values"), (dict(steps=60, coefficients=(1.2, 0.0, 0.0)), "singular values"),
                                     (dict(momentum=None), "momentum"), (dict(momentum=float("nan")), "momentum"), (dict(weight_decay="much"), "weight_decay")])
def test_settings_that_no_step_takes_are_refused_by_the_constructor(train, bad, why):  # noqa: F811
    with pytest.raises(ValueError, match=why):
        train.RenderTrainer({"network_fn": nets(1)[0]}, muon=bad)


def test_other_settings_are_taken_as_they_are(train):  # noqa: F811
    t = train.RenderTrainer({"network_fn": nets(1)[0]}, muon=dict(coefficients=[1.5, -0.5, 0.0], steps=12, scale="none", precision="fp16", nesterov=False, momentum=0))
    assert t.muon["coefficients"] == (1.5, -0.5, 0.0) and t.muon["steps"] == 12 and t.muon["momentum"] == 0.0 and t.muon["nesterov"] is False
    set_grads(t.nets, 1)
    t.apply_gradients()
    assert t.opt_step == 1
