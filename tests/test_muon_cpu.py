"""CPU: what orthogonalise, muon_step_ and adam_step_multi_ refuse, on the host and before any device work; workspace sizes."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def S():
    import spin_nerf_amd as S
    S._lib.load()
    return S


def test_orthogonalise_refusals(S):
    x = torch.zeros(4, 4)
    for bad, why in [(torch.zeros(4), "expected a tensor"), (torch.zeros(4, 4, dtype=torch.float64), "float32, float16"),
                     (torch.zeros(4, 4, dtype=torch.int32), "float32, float16"), (3.0, "expected a tensor")]:
        with pytest.raises(ValueError, match=why):
            S.orthogonalise(bad)
    for kw, why in [(dict(steps=0), "steps"), (dict(steps=101), "steps"), (dict(steps=2.5), "steps"), (dict(eps=0.0), "eps"),
                    (dict(eps=float("nan")), "eps"), (dict(precision="bf16"), "precision")]:
        with pytest.raises(ValueError, match=why):
            S.orthogonalise(x, **kw)
    with pytest.raises(RuntimeError, match="no backward"):
        S.orthogonalise(x.clone().requires_grad_())
    with pytest.raises(S.HipLibraryError, match="CPU tensor"):
        S.orthogonalise(x)


def test_muon_and_adam_refusals(S):
    a, b, c = torch.zeros(4, 4), torch.zeros(4, 4), torch.zeros(4, 4)
    with pytest.raises(S.HipLibraryError, match="CPU tensor"):
        S.muon_step_([a], [b], [c], 1e-3)
    with pytest.raises(ValueError, match="length"):
        S.muon_step_([a], [b, b], [c], 1e-3)
    with pytest.raises(ValueError, match="scale"):
        S.muon_step_([a], [b], [c], 1e-3, scale="adam")
    with pytest.raises(ValueError, match="precision"):
        S.muon_step_([a], [b], [c], 1e-3, precision=None)
    with pytest.raises(S.HipLibraryError, match="CPU tensor"):
        S.adam_step_multi_([a], [b], [c], [a], 1e-3, 1)


def test_entry_points_refuse_before_any_device_access(S):
    lib, L = S._lib.load(), S._lib
    one = ctypes.c_void_p(256)

    def orth(x=one, dt=0, batch=1, m=8, n=8, out=one, ob=64, orow=8, steps=5, co=(3.4445, -4.775, 2.0315), eps=1e-7, prec=0, ws=one):
        return lib.snr_orthogonalise(x, dt, batch, m, n, 64, 8, out, ob, orow, steps, *co, eps, prec, ws, None)
    assert orth(x=None) == -1 and orth(out=None) == -1 and orth(ws=None) == -1
    for kw in (dict(m=0), dict(n=0), dict(batch=0), dict(batch=1 << 17), dict(m=1 << 17), dict(steps=0), dict(steps=101), dict(eps=0.0),
               dict(eps=float("nan")), dict(orow=7), dict(batch=2, ob=63)):
        assert orth(**kw) == -2, kw
    for kw in (dict(dt=3), dict(prec=2), dict(co=(16.0, 0.0, 0.0)), dict(co=(1.0, 100.0, 0.0)), dict(co=(float("nan"), 0.0, 0.0))):
        assert orth(**kw) == -3, kw
    items = (L.MuonItem * 2)()

    def muon(items=items, n=1, mode=1, ws=one, co=(3.4445, -4.775, 2.0315)):
        return lib.snr_muon_step_multi(items, n, 1e-3, 0.95, 1, 0.0, mode, 5, *co, 1e-7, 1.0, 0, None, ws, None)
    assert muon(items=None) == -1 and muon(ws=None) == -1 and muon(n=0) == -2 and muon(mode=3) == -3 and muon() == -1
    items[0] = L.MuonItem(256, 256, 256, 1, 0, 4)
    assert muon() == -2 and muon(co=(9.0, 0.0, 0.0)) == -3
    ad = (L.AdamItem * 1)()
    adam = lambda it=ad, n=1, step=1: lib.snr_adam_step_multi(it, n, 1e-3, 0.9, 0.999, 1e-8, step, 1.0, None, None)   # noqa: E731
    assert adam(it=None) == -1 and adam(n=0) == -2 and adam(step=0) == -2
    ad[0] = L.AdamItem(None, None, None, None, 4)
    assert adam() == -1
    ad[0] = L.AdamItem(256, 256, 256, 256, -1)
    assert adam() == -2


def test_workspace_sizes(S):
    lib, L = S._lib.load(), S._lib
    one = lib.snr_orthogonalise_ws_bytes(1, 256, 256, 0)
    least = 3 * 256 * 256 * 2      # X in 22 bits and the Gram matrix
    assert one >= least and lib.snr_orthogonalise_ws_bytes(4, 256, 256, 0) >= 4 * least
    assert lib.snr_orthogonalise_ws_bytes(1, 256, 319, 1) == lib.snr_orthogonalise_ws_bytes(1, 319, 256, 1) > one
    assert lib.snr_orthogonalise_ws_bytes(0, 8, 8, 0) == -2 and lib.snr_orthogonalise_ws_bytes(1, 8, 8, 5) == -3
    assert lib.snr_orthogonalise_ws_bytes(1, 65536, 65536, 1) > 1 << 34          # sizes are 64-bit
    it = (L.MuonItem * 30)(*[L.MuonItem(256, 256, 256, 1, 64, 64)] * 30)
    assert lib.snr_muon_ws_bytes(it, 1, 0) > 0 and lib.snr_muon_ws_bytes(it, 30, 0) >= lib.snr_muon_ws_bytes(it, 2, 0)
    assert lib.snr_muon_ws_bytes(None, 1, 0) == -1 and lib.snr_muon_ws_bytes(it, 0, 0) == -2


def test_launches_past_the_largest_grid_are_refused(S):
    """a launch holds fewer than 2^32 threads: 2^22 workgroups of up to 1024, 2^24 of 256 (each with 1024 of Adam's values)"""
    lib, L = S._lib.load(), S._lib
    assert lib.snr_orthogonalise_ws_bytes(65536, 1, 65536, 0) == -2              # 1024 tiles a matrix
    assert lib.snr_orthogonalise_ws_bytes(4096, 1, 65536, 0) > 0
    it = (L.MuonItem * 2)(L.MuonItem(256, 256, 256, 4096, 1, 65536), L.MuonItem(256, 256, 256, 1, 1, 65536))
    assert lib.snr_muon_ws_bytes(it, 1, 0) > 0 and lib.snr_muon_ws_bytes(it, 2, 0) == -2
    ad = (L.AdamItem * 1)(L.AdamItem(256, 256, 256, 256, 1 << 34))
    assert lib.snr_adam_step_multi(ad, 1, 1e-3, 0.9, 0.999, 1e-8, 1, 1.0, None, None) == -2
