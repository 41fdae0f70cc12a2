"""muon_update writes parameters and momenta in place: no two of them may share memory, nor a gradient with either
(checks come before any GPU call, so these run without one)."""
import pytest
import torch

from nerfhip import _lib, muon


def test_shared_memory_is_refused():
    whole = torch.zeros(3 * 24)
    a, b, c = whole[:24].view(4, 6), whole[24:48].view(4, 6), whole[48:].view(4, 6)
    across = whole[12:36].view(4, 6)        # half of a, half of b
    new = lambda: torch.zeros(4, 6)
    for p, g, m in (([a, across], [new(), new()], [new(), new()]), ([a], [new()], [across]),
                    ([a], [a], [new()]), ([a], [new()], [a]), ([new()], [b], [b]), ([a], [across], [new()]),
                    ([new()], [across], [b]), ([a, b], [new(), across], [new(), new()])):
        with pytest.raises(ValueError, match="muon_update"):
            muon.muon_update(p, g, m, 0.1)
    # neighbours in one allocation, and one gradient for two matrices, are fine (and get as far as the device)
    for p, g, m in (([a], [b], [c]), ([a, b], [c, c], [new(), new()]),
                    ([a], [whole[24:48].view(4, 6)], [new()])):
        with pytest.raises(_lib.NerfHipError, match="ROCm GPU"):
            muon.muon_update(p, g, m, 0.1)
