"""eps reaches the kernels as a 32-bit number: what is none, or rounds to zero or infinity, is refused (before any GPU
call, so these run without one)."""
import pytest
import torch

from nerfhip import _lib, muon


@pytest.mark.parametrize("eps", [0.0, -1.0, 1e-50, 1e39, float("inf"), float("nan")])
def test_eps_that_is_no_positive_32_bit_number(eps):
    p = torch.zeros(4, 6)
    with pytest.raises(ValueError, match="eps"):
        muon.orthogonalize(p, eps=eps)
    with pytest.raises(ValueError, match="eps"):
        muon.muon_update([p], [p.clone()], [p.clone()], 0.1, eps=eps)


@pytest.mark.parametrize("eps", [1e-45, 1e-30, 1e38])
def test_other_eps_get_as_far_as_the_device(eps):
    with pytest.raises(_lib.NerfHipError, match="ROCm GPU"):
        muon.orthogonalize(torch.zeros(4, 6), eps=eps)
