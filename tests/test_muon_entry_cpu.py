"""CPU: calls of the C entries whose launches would get in each other's way are refused before the first of them."""
import pytest

SHAPE, UNSUPPORTED = -2, -3


@pytest.fixture(scope="module")
def L():
    import spin_nerf_amd as S
    S._lib.load()
    return S._lib


def test_out_is_x_or_shares_nothing_with_a_stack(L):
    """(the pointers are numbers, and no call gets past the precision, which is checked behind the overlap)"""
    lib = L.load()

    def orth(x, out, batch=4, m=8, n=8, xb=64, xr=8, ob=64, orow=8, dt=0):
        return lib.snr_orthogonalise(x, dt, batch, m, n, xb, xr, out, ob, orow, 5, 3.4445, -4.775, 2.0315, 1e-7, 9, 1 << 30, None)
    at = 1 << 20
    whole = 4 * 64 * 4
    for x, out, kw in ((at, at + 256, {}), (at + 256, at, {}), (at, at + whole - 4, {}), (at, at - whole + 4, {}),   # shifted by less than the stack
                       (at, at, dict(xb=72)), (at, at, dict(xr=16, xb=128)), (at, at, dict(xb=0)),                  # the same place, other strides
                       (at, at + whole // 2 - 2, dict(dt=1)), (at, at + 8, dict(batch=2, m=1, n=3, xb=3, xr=3, ob=3, orow=3))):
        assert orth(x, out, **kw) == SHAPE, (x - at, out - at, kw)
    for x, out, kw in ((at, at, {}), (at, at + whole, {}), (at, at - whole, {}), (at, at + whole // 2, dict(dt=1)),
                       (at, at, dict(m=1, n=64, xr=8, orow=64)), (at, at, dict(m=1, n=64, xr=100, orow=64)),      # one row: its stride says nothing
                       (at, at + 32, dict(batch=1)), (at, at, dict(batch=1, xb=7))):                                # one matrix is read before it is written
        assert orth(x, out, **kw) == UNSUPPORTED, (x - at, out - at, kw)


def test_a_step_that_is_refused_has_not_begun(L):
    """300 matrices of 8 x 8 are a launch of their own, ahead of the 4097 whose grid would be too large"""
    lib = L.load()
    small, large = L.MuonItem(1 << 20, 1 << 24, 1 << 28, 300, 8, 8), L.MuonItem(1 << 40, 1 << 42, 1 << 44, 4097, 1, 65536)

    def muon(items):
        return lib.snr_muon_step_multi((L.MuonItem * len(items))(*items), len(items), 1e-3, 0.95, 1, 0.0, 1, 5, 3.4445, -4.775, 2.0315, 1e-7, 1.0,
                                       0, None, 1 << 30, None)
    assert muon([large]) == SHAPE and muon([small, large]) == SHAPE and muon([large, small]) == SHAPE
