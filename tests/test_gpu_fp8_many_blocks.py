"""Weights of more blocks than one launch has threads for (2^24 blocks of 256 threads)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev():
    if torch.cuda.mem_get_info()[0] < 32 << 30:
        pytest.skip("needs 32 GB")
    return torch.device("cuda:0")


def same(a, b):
    return torch.equal(a.q.view(torch.uint8), b.q.view(torch.uint8)) and torch.equal(a.scale, b.scale)


def test_many_small_matrices(dev):
    from nerfhip import fp8
    E = (1 << 24) + 301
    w = torch.empty(E, 1, 2, device=dev).normal_(generator=torch.Generator(device=dev).manual_seed(1))
    f = fp8.quantize_weight(w)
    for lo in (0, 1 << 23, (1 << 24) - 5, E - 300):
        assert same(fp8.Fp8Weight(f.q[lo:lo + 300], f.scale[lo:lo + 300], 2), fp8.quantize_weight(w[lo:lo + 300])), lo
    top = w.abs().amax((1, 2))
    assert bool((f.scale.flatten() > 0).all()) and bool((f.q[:, :, :2].float().abs().amax((1, 2)) > 200).all())
    back = torch.ldexp(f.q[:, 0, :2].float(), f.scale.view(-1, 1).int() - 127)
    assert float(((back - w[:, 0]).abs() / top[:, None]).max()) <= 2.0 ** -4
