"""GPU: orthogonalise and muon_step_ where the large tiles, and a table of many sizes, do the work; tolerances as in
test_gpu_muon.py, whose oracle and bounds these tests use (few steps: the oracle's products are on the CPU)."""
import pytest
import torch

from test_gpu_muon import HALF, NS, bound32, check, gradient_like, muon_case, muon_oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def S():
    import spin_nerf_amd as S
    return S


# tiles of 128: 135 symmetric ones of 3 x 1100; of 192 and 256: 300 and 320 of 20 x 900; one matrix whose rows pass 1000 chunks of the norm
@pytest.mark.parametrize("shape", [(3, 1100, 1500), (20, 900, 901), (3, 1500, 1100), (20, 905, 900), (2100, 4100)])
@pytest.mark.parametrize("precision", ["fp32", "fp16"])
def test_large_tiles_match_the_formula(S, shape, precision):
    x = gradient_like(torch.Generator().manual_seed(shape[-1]), *shape)
    steps = 2 if len(shape) == 3 else 1
    for dtype in (torch.float32, torch.bfloat16):
        got = S.orthogonalise(x.to(dtype).cuda(), steps=steps, precision=precision)
        check(got, x.to(dtype), precision, steps)


@pytest.mark.parametrize("precision", ["fp32", "fp16"])
@pytest.mark.parametrize("shapes", [[(20, 900, 901)], [(3, 1500, 1100), (96, 128)],
                                    [(70, 70), (70, 100), (2, 90, 71), (100, 70), (129, 128), (200, 65), (66, 67), (256, 319), (3, 150, 300)]])
def test_muon_with_large_tiles_and_with_many_sizes(S, shapes, precision):
    lr, mu, wd = 0.02, 0.95, 0.1
    p, g, m = muon_case(torch.Generator().manual_seed(21), shapes)
    dp, dg, dm = ([t.cuda() for t in ts] for ts in (p, g, m))
    S.muon_step_(dp, dg, dm, lr, momentum=mu, weight_decay=wd, precision=precision, steps=2)
    for P, G, M, gp, gm in zip(p, g, m, dp, dm):
        rp, rm, step, o, norms = muon_oracle(P, G, M, lr, mu, True, wd, "spectral", 1.0, steps=2)
        assert float((gm.cpu().double() - rm).norm()) <= 3 * 2.0 ** -24 * float(rm.norm() + G.double().norm())
        off, size = (gp.cpu().double() - rp).flatten(-2).norm(dim=-1), o.flatten(-2).norm(dim=-1)
        # as for the small ones; two steps amplify the momentum's roundings by at most 3.4445^2 < 12
        tol = step * ((HALF * size if precision == "fp16" else bound32(norms, 2, NS[0])) + 12 * 4 * 2.0 ** -24) \
            + 4 * 2.0 ** -24 * P.double().flatten(-2).norm(dim=-1)
        assert bool((off <= tol).all()), (float(off.max()), float(tol.min()))


# what one workgroup keeps: 64 x 448 and 128 x 128 at fp32's accuracy, 128 x 320 with fp16 products; both sides of each edge
@pytest.mark.parametrize("m,n", [(64, 65), (65, 65), (66, 129), (128, 128), (129, 128), (128, 192), (193, 128), (100, 319), (320, 128), (70, 321), (448, 64)])
@pytest.mark.parametrize("precision", ["fp32", "fp16"])
def test_sizes_around_what_one_workgroup_keeps(S, m, n, precision):
    gen = torch.Generator().manual_seed(m + n)
    for dtype in (torch.float32, torch.bfloat16):
        x = gradient_like(gen, 2, m, n).to(dtype)
        check(S.orthogonalise(x.cuda(), precision=precision), x, precision)
    p, g, b = muon_case(gen, [(3, m, n), (n, m)])
    dp, dg, db = ([t.cuda() for t in ts] for ts in (p, g, b))
    S.muon_step_(dp, dg, db, 0.02, weight_decay=0.1, precision=precision)
    for P, G, M, gp, gm in zip(p, g, b, dp, db):
        rp, rm, step, o, norms = muon_oracle(P, G, M, 0.02, 0.95, True, 0.1, "spectral", 1.0)
        assert float((gm.cpu().double() - rm).norm()) <= 3 * 2.0 ** -24 * float(rm.norm() + G.double().norm())
        off, size = (gp.cpu().double() - rp).flatten(-2).norm(dim=-1), o.flatten(-2).norm(dim=-1)
        tol = step * ((HALF * size if precision == "fp16" else bound32(norms, 5, NS[0])) + 485 * 4 * 2.0 ** -24) \
            + 4 * 2.0 ** -24 * P.double().flatten(-2).norm(dim=-1)
        assert bool((off <= tol).all()), (float(off.max()), float(tol.min()))


@pytest.mark.parametrize("n", [1, 33, 64, 100, 300])
def test_diagonal_and_mostly_empty_matrices(S, n):
    """a diagonal one keeps its zeros exactly, in either precision: no product of two different rows has a nonzero term"""
    d = torch.diag(torch.linspace(0.5, 2.0, n))
    for precision in ("fp32", "fp16"):
        got = S.orthogonalise(d.cuda(), precision=precision).cpu()
        assert bool((got[~torch.eye(n, dtype=torch.bool)] == 0).all())
        check(got, d, precision)
    one = torch.zeros(n, n + 3)
    one[n // 2, n // 3] = -3.0                       # a single entry: s = 1 all along
    got = S.orthogonalise(one.cuda()).cpu()
    check(got, one, "fp32")
    assert int((got != 0).sum()) == 1


def test_a_matrix_gives_the_same_bits_alone_and_in_company(S):
    """(to the bit while the calls take the same tiles, which go by how much work there is)"""
    gen = torch.Generator().manual_seed(4)
    x = gradient_like(gen, 6, 200, 300).cuda()
    many = S.orthogonalise(x)
    for k in (0, 5):
        assert torch.equal(S.orthogonalise(x[k]), many[k])


def test_largest_batch_of_the_smallest(S):
    x = torch.randn(65536, 2, 3, generator=torch.Generator().manual_seed(5))
    got = S.orthogonalise(x.cuda())
    check(got, x, "fp32")
    with pytest.raises(S.HipLibraryError, match="size"):
        S.orthogonalise(torch.zeros(65537, 1, 1, device="cuda"))
