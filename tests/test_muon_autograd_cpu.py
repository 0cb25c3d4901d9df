"""CPU: orthogonalise has no derivative, neither backward nor forward mode, and says so before any device work."""
import pytest
import torch
import torch.autograd.forward_ad as fwd


def test_a_tangent_is_refused_not_dropped():
    import spin_nerf_amd as S
    x, t = torch.randn(4, 5), torch.randn(4, 5)
    with fwd.dual_level():
        dual = fwd.make_dual(x, t)
        for call in (lambda: S.orthogonalise(dual), lambda: S.orthogonalise(dual.mT), lambda: S.orthogonalise(x, out=fwd.make_dual(torch.empty(4, 5), t))):
            with pytest.raises(RuntimeError, match="forward"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward"):     # (no_grad leaves forward mode on)
                call()
        with pytest.raises(S.HipLibraryError, match="CPU tensor"):                  # its primal alone is a tensor like any other
            S.orthogonalise(fwd.unpack_dual(dual).primal)
        with pytest.raises(S.HipLibraryError, match="CPU tensor"):
            S.orthogonalise(x)
