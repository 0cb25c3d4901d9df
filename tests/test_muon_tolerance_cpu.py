"""CPU: the tolerances of the GPU tests of orthogonalise tell a kernel that loses a plane from one that does not."""
import pytest
import torch

from muon_emulation import NS, bound, emulate, gradient_like, oracle


@pytest.mark.parametrize("shape,steps", [((66, 65), 5), ((128, 283), 5), ((2, 250, 300), 5), ((300, 250), 2), ((500, 512), 1), ((1, 700, 900), 2)])
def test_the_tolerances_tell_a_lost_plane(shape, steps):
    x = gradient_like(shape, 7)
    ref = oracle(x, steps)
    whole, halves, lost = ((emulate(x, steps, NS, *how) - ref).flatten(-2).norm(dim=-1) for how in ((True, True), (False, True), (False, False)))
    for precision, right, wrong in (("fp32", whole, halves), ("fp16", halves, lost)):
        tol = bound(x, ref, steps, precision)
        assert bool((2 * right < tol).all()) and bool((2 * tol < wrong).all()), (precision, right / tol, wrong / tol)
    assert float(whole.max()) < 2e-6 * float(ref.norm())      # (planes of 22 bits: about what 32-bit products do)


def test_what_the_quintic_does_to_singular_values():
    """no value from [0, 1] is ever lifted past 1.21, and five steps bring what was above 0.003 to 0.66 or more"""
    s = torch.linspace(0, 1, 200001, dtype=torch.float64)
    x = s
    for _ in range(5):
        x = x * (NS[0] + NS[1] * x * x + NS[2] * x ** 4)
        assert 1.19 < float(x.max()) < 1.21
    assert 0.66 < float(x[s > 0.003].min()) < 0.7
