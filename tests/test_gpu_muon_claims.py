"""GPU: what the documentation of orthogonalise says of single matrices holds in a stack that goes through tiles too, and in stacks whose
offsets pass 32 bits."""
import pytest
import torch

from muon_emulation import NS, bound, gradient_like, oracle

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


@pytest.fixture(scope="module")
def S():
    import spin_nerf_amd as S
    return S


def norm(x):
    return x.double().flatten(-2).norm(dim=-1)


@pytest.mark.parametrize("precision", ["fp32", "fp16"])
@pytest.mark.parametrize("shape,steps", [((9, 70, 90), 5), ((9, 250, 300), 5), ((9, 300, 251), 5), ((20, 1000, 1030), 1), ((20, 1030, 1000), 1)])
def test_a_matrix_that_is_zero_tiny_huge_or_not_finite_is_alone_with_it(S, shape, steps, precision):
    x = gradient_like(shape, 3)
    x[1] = 0
    x[2] *= 1e33                                   # squares pass fp32
    x[3, 3, 4] = float("nan")
    x[4, -1, -1] = float("inf")
    x[5, 0, -1] = float("-inf")
    x[6] *= 1e-30                                  # a norm below eps: x / eps, nearly nothing
    x = x.cuda()
    got = S.orthogonalise(x, steps=steps, coefficients=NS, precision=precision)
    for k in (3, 4, 5):
        assert bool(torch.isnan(got[k]).all())
    # |x| / eps < 1e-23 times a^5 = 485.  In tiles it is nothing at all: 1024 x / eps is below 1e-21 an entry, and the planes' least
    # value is 2^-24 / 2048 = 2.9e-11
    assert bool((got[1] == 0).all()) and float(got[6].abs().max()) < 1e-18
    fine = [0, 2, 7, 8]
    z = x[fine].clone()
    z[1] = gradient_like(shape, 3)[2].cuda()       # (the formula's sums in 64 bits have no trouble; the emulation's norm neither)
    ref = oracle(z, steps)
    tol = bound(z, ref, steps, precision) + 2 * EPS * norm(ref)          # (x[2] was rounded once more)
    assert bool((norm(got[fine] - ref) <= tol).all())
    # ... and in an optimizer step: its parameters and its momentum alone
    p, m = torch.zeros_like(x), torch.zeros_like(x)
    S.muon_step_([p], [x], [m], 1.0, nesterov=False, scale="none", steps=steps, coefficients=NS, precision=precision)
    assert bool((norm(p[fine] + ref) <= tol + EPS * norm(ref)).all()) and bool(torch.isnan(p[3:6]).flatten(1).all(1).all()) and bool((p[1] == 0).all())


def test_offsets_past_32_bits_one_workgroup_a_matrix(S):
    """65536 matrices of 128 x 300 bf16: 2.5e9 values in and out"""
    x = torch.empty(65536, 128, 300, device="cuda", dtype=torch.bfloat16)
    some = gradient_like((6, 128, 300), 4).bfloat16().cuda()
    for k in range(0, 65536, 4096):
        x[k:k + 4096] = some[0]
    at = [0, 1, 32768, 55924, 55925, 65535]        # 2^31 values lie at matrix 55924.05
    x[at] = some
    got = S.orthogonalise(x)
    want = S.orthogonalise(some)
    assert torch.equal(got[at], want) and torch.equal(got[65534], want[0]) and torch.equal(got[55923], want[0])
    S.orthogonalise(x, out=x)
    assert torch.equal(x[at], want) and torch.equal(x[4000], want[0])


@pytest.mark.parametrize("precision", ["fp32", "fp16"])
def test_offsets_past_32_bits_in_tiles(S, precision):
    """2100 matrices of 1030 x 1000 fp32: 2.2e9 values, and more of their planes"""
    x = torch.empty(2100, 1030, 1000, device="cuda")
    some = gradient_like((5, 1030, 1000), 5).cuda()
    x[:] = some[0]
    at = [0, 7, 2084, 2085, 2099]                  # 2^31 values lie at matrix 2084.9
    x[at] = some
    S.orthogonalise(x, steps=1, coefficients=NS, precision=precision, out=x)
    ref = oracle(some, 1)
    tol = bound(some, ref, 1, precision) + EPS * norm(ref)
    assert bool((norm(x[at] - ref) <= tol).all())
    for k in (1, 2083, 2098):
        assert torch.equal(x[k], x[1000])
