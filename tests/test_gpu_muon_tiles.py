"""GPU: every kernel of orthogonalise and muon_step_ against the formula in 64 bits, at sizes that reach it (test_muon_tiles_cpu.py holds
them to that) and with tolerances that see a plane that is lost (muon_emulation.py: bound).  Inputs and results are fp32, whose own
rounding is 2^-24 a value."""
import pytest
import torch

from muon_emulation import LISTS, NS, ONE, TILED, bound, gradient_like, oracle, steps_for

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


@pytest.fixture(scope="module")
def S():
    import spin_nerf_amd as S
    return S


def norm(x):
    return x.double().flatten(-2).norm(dim=-1)


@pytest.mark.parametrize("precision", ["fp32", "fp16"])
@pytest.mark.parametrize("shape", ONE + TILED)
def test_orthogonalise(S, shape, precision):
    steps = steps_for(shape)
    x = gradient_like(shape, sum(shape)).cuda()
    # where the shorter side is 64 or less, fp16 asks for fp32's accuracy too
    ref, how = oracle(x, steps), "fp32" if min(shape[-2:]) <= 64 else precision
    tol = bound(x, ref, steps, how) + EPS * norm(ref)
    off = norm(S.orthogonalise(x, steps=steps, coefficients=NS, precision=precision) - ref)
    assert bool((off <= tol).all()), (off / norm(ref), tol / norm(ref))
    # off the 16-byte grid: the other way of reading and (in place) of writing
    buf = torch.full((x.numel() + 8,), 7.0, device="cuda")
    y = buf[3:3 + x.numel()].view(x.shape)
    y.copy_(x)
    S.orthogonalise(y, steps=steps, coefficients=NS, precision=precision, out=y)
    assert bool((norm(y - ref) <= tol).all()) and bool((buf[:3] == 7).all()) and bool((buf[3 + x.numel():] == 7).all())


@pytest.mark.parametrize("precision", ["fp32", "fp16"])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("shapes", LISTS)
def test_muon_step(S, shapes, shift, precision):
    """rate 1 and scale "none": what the parameters move by is the orthogonalised matrix itself"""
    wd, steps = 0.1, min(steps_for(s) for s in shapes)
    g = [gradient_like(s, sum(s) + 1).cuda() for s in shapes]
    flat = torch.rand(sum(t.numel() for t in g) + 8, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) * 0.2 - 0.1
    p, o = [], shift
    for t in g:                                    # (shift 1: parameters off the 16-byte grid)
        p.append(flat[o:o + t.numel()].view(t.shape))
        o += t.numel()
    before, m = flat.clone(), [torch.zeros_like(t) for t in g]
    start = [t.clone() for t in p]
    S.muon_step_(p, g, m, 1.0, nesterov=False, weight_decay=wd, scale="none", steps=steps, coefficients=NS, precision=precision)
    for s, P, P0, G, M in zip(shapes, p, start, g, m):
        assert torch.equal(M, G)                   # momentum from zero: the update is the gradient
        ref, how = oracle(G, steps), "fp32" if min(s[-2:]) <= 64 else precision
        # 1 - lr wd, its product, the rate's and the difference: a rounding each
        tol = bound(G, ref, steps, how) + 2 * EPS * norm(ref) + 3 * EPS * norm(P0)
        off = norm(P.double() - (P0.double() * (1 - wd) - ref))
        assert bool((off <= tol).all()), (s, off / norm(ref), tol / norm(ref))
    assert torch.equal(flat[:shift], before[:shift]) and torch.equal(flat[o:], before[o:])
