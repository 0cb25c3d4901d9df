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
