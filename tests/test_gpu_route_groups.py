"""The gate's choice of groups where their keys are larger than their scores: 32 bits do not decide it. Choices have
to be equal to those of 64 bits on the CPU."""
import pytest
import torch

from test_gpu_experts import ref_choice, ref_scores

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


def chosen(dev, x, k, score="softmax", bias=None, groups=1, top_groups=1, group_score="max"):
    from nerfhip import experts
    w, e = experts.route(x.to(dev), k, score=score, bias=None if bias is None else bias.to(dev), groups=groups,
                         top_groups=top_groups, group_score=group_score)
    return w.cpu(), e.cpu().long()


@pytest.mark.parametrize("B", [0.7, 64.0, 1024.0, 1e5, 1e6])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E", [4, 64, 512])
def test_groups_whose_two_highest_keys_cancel(dev, B, score, E):
    """Each group's two highest keys are near +B and -B (the others far below): the sums are small, the keys'
    own rounding is not."""
    T, per = (200000, 2) if E == 4 else (20000, 16)
    g = torch.Generator().manual_seed(int(B) + E)
    x = torch.randn(T, E, generator=g)
    bias = torch.full((E,), -8.0 * B)
    bias[0::per], bias[1::per] = B, -B
    want = ref_choice(x, 1, score, bias, E // per, 1, "top2")
    _, e = chosen(dev, x, 1, score, bias, E // per, 1, "top2")
    assert torch.equal(e // per, want // per)
    assert torch.equal(e, want)


def test_nearly_tied_groups_of_a_softmax(dev):
    """512 experts, pairs of groups whose sums of about +0.7 and -0.7 differ by less than a key's step."""
    T, E, per = 20000, 512, 16
    g = torch.Generator().manual_seed(5)
    x = torch.randn(1, E, generator=g)
    s = ref_scores(x, "softmax")[0]
    bias = torch.full((E,), -50.0)
    bias[0::per] = (0.7 - s[0::per]).float()
    bias[1::per] = (-0.7 - s[1::per]).float()
    x = x + 1e-4 * torch.randn(T, E, generator=g)
    want = ref_choice(x, 2, "softmax", bias, E // per, 1, "top2")
    _, e = chosen(dev, x, 2, "softmax", bias, E // per, 1, "top2")
    assert torch.equal(e, want)


def test_a_large_group_below_the_first_one_dropped(dev):
    """In 32 bits the third group lies below the second by less than its own (large) keys' step."""
    T, per, B = 50000, 2, 3e6
    g = torch.Generator().manual_seed(6)
    x = torch.randn(T, 6, generator=g)
    bias = torch.tensor([0.5, 0.0, 0.48, 0.0, B, 0.5 - B])
    want = ref_choice(x, 1, "sigmoid", bias, 3, 1, "top2")
    _, e = chosen(dev, x, 1, "sigmoid", bias, 3, 1, "top2")
    assert torch.equal(e, want)
