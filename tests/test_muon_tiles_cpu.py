"""CPU: the sizes at which the GPU tests compare orthogonalise and muon_step_ with the formula reach every kernel, whatever becomes of the rules."""
import ctypes

import pytest
import torch

from muon_emulation import LISTS, ONE, TILED


@pytest.fixture(scope="module")
def L():
    import spin_nerf_amd as S
    S._lib.load()
    return S._lib


def routes(L, shapes, precision):
    items = [L.MuonItem(256, 256, 256, *((1,) * (3 - len(s)) + tuple(s))) for s in shapes]
    out = (ctypes.c_int * 30)()
    n = L.load().snr_muon_routes((L.MuonItem * len(items))(*items), len(items), precision, out, 10)
    assert 0 < n <= 10
    return [tuple(out[3 * i:3 * i + 3]) for i in range(n)]


TILES, TILES_FP16 = 8, 9


def test_the_sizes_reach_every_kernel(L):
    if torch.cuda.is_available() and torch.cuda.get_device_properties(0).multi_processor_count != 256:
        pytest.skip("tiles go by the number of compute units")
    kinds = {r[0] for p in (0, 1) for s in ONE for r in routes(L, [s], p)}
    assert kinds >= set(range(TILES)), kinds
    for what in (TILED, [s for q in LISTS for s in q]):
        taken = [(r, s[-2] > s[-1]) for p in (0, 1) for s in what for r in routes(L, [s], p) if r[0] >= TILES]
        assert {r[:2] for r, _ in taken} == {(TILES, t) for t in (32, 64, 128)} | {(TILES_FP16, t) for t in (32, 64, 128, 192)}
        for tall in (False, True):           # (a matrix and its transpose end differently)
            assert {(r[0], r[2]) for r, t in taken if t == tall} == {(TILES, t) for t in (32, 64, 128)} | {(TILES_FP16, t) for t in (32, 64, 128, 256)}
    # the two networks' list goes as one sequence, whose symmetric tiles are 64 wide
    assert routes(L, LISTS[-1], 0) == [(TILES_FP16, 64, 64)] and routes(L, LISTS[-1], 1) == [(TILES, 64, 64)]


def test_routes_refuse_what_the_step_refuses(L):
    lib, it = L.load(), (L.MuonItem * 1)(L.MuonItem(256, 256, 256, 1, 8, 8))
    out = (ctypes.c_int * 3)()
    assert lib.snr_muon_routes(None, 1, 0, out, 1) == -1 and lib.snr_muon_routes(it, 1, 0, None, 1) == -1
    assert lib.snr_muon_routes(it, 0, 0, out, 1) == -2 and lib.snr_muon_routes(it, 1, 2, out, 1) == -3
    assert lib.snr_muon_routes(it, 1, 0, None, 0) == 1 and lib.snr_muon_routes(it, 1, 0, out, 1) == 1 and list(out) == [0, 0, 0]
