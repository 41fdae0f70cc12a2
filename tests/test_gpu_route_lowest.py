"""Masks of the type's lowest value beside masks of minus infinity, and group scores beyond 32 bits' range: choices
have to be equal to those of 64 bits on the CPU."""
import math

import pytest
import torch

from test_gpu_experts import ref_scores

pytestmark = pytest.mark.gpu

INF, LOW = math.inf, torch.finfo(torch.float32).min


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


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_the_lowest_value_goes_before_minus_infinity(dev, score):
    x = torch.full((4, 20), -INF)
    x[0, 5] = LOW
    x[1, 3], x[1, 9], x[1, 17] = LOW, 1.0, LOW
    x[2, 1:] = LOW
    x[3, 19] = LOW
    x[3, 4] = math.nan
    w, e = chosen(dev, x, 3, score)
    assert e[0].tolist() == [5, 0, 1] and e[1].tolist() == [9, 3, 17] and e[2].tolist() == [1, 2, 3]
    assert e[3].tolist() == [19, 0, 1]
    assert w[0].tolist() == [1.0, 0.0, 0.0] and w[1].tolist() == [1.0, 0.0, 0.0]
    assert torch.allclose(w[2], torch.full((3,), 1 / 3)) and bool(torch.isnan(w[3]).all())
    # groups of 5: rows 0 and 3 keep the one that holds an expert
    _, e = chosen(dev, x[:1], 2, score, groups=4, top_groups=1)
    assert e[0].tolist() == [5, 6]


@pytest.mark.parametrize("E,groups", [(20, 1), (64, 1), (300, 1), (20, 5), (64, 8), (300, 30)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_biases_of_the_lowest_value_and_minus_infinity(dev, E, groups, score):
    """Biases of -inf, of the lowest value and ordinary ones, in random places: ordinary experts first, then
    the lowest in order of their index, then the forbidden ones."""
    g = torch.Generator().manual_seed(E + groups)
    for _ in range(20):
        x = torch.randn(50, E, generator=g)
        kind = torch.randint(0, 3, (E,), generator=g)
        bias = 0.1 * torch.randn(E, generator=g)
        bias = torch.where(kind == 1, torch.full_like(bias, LOW), torch.where(kind == 2, torch.full_like(bias, -INF), bias))
        top = max(1, groups // 2)
        k = min(32, top * (E // groups))
        for gs in ("max", "top2") if groups > 1 else ("max",):
            want = exact_choice(ref_scores(x, score) + bias.double(), k, groups, top, gs)
            _, e = chosen(dev, x, k, score, bias, groups, top, gs)
            assert torch.equal(e, want), (E, groups, gs)


def exact_choice(key, k, groups, top_groups, group_score):
    """By Python's own sorting of tuples: 64-bit keys, -inf below every number."""
    out = []
    for row in key.tolist():
        per = len(row) // groups
        score = []
        for j in range(groups):
            best = sorted(row[j * per:(j + 1) * per], reverse=True)
            score.append(sum(best[:2]) if group_score == "top2" else best[0])
        kept = sorted(range(groups), key=lambda j: (-score[j], j))[:top_groups]
        left = [i for j in kept for i in range(j * per, (j + 1) * per)]
        out.append(sorted(left, key=lambda i: (-row[i], i))[:k])
    return torch.tensor(out)


def test_keys_beyond_the_range_of_32_bits(dev):
    """Group scores whose 32-bit sum overflows either way: 64 bits tell them apart."""
    big = torch.finfo(torch.float32).max
    x = torch.zeros(3, 8)
    for bias, first in ((torch.tensor([big, big, big, 0.0, big, big / 2, 0.0, 0.0]), 0),
                        (torch.tensor([big, big / 2, big, big, 0.0, 0.0, 0.0, 0.0]), 2),
                        (torch.tensor([LOW, LOW, LOW / 2, LOW, -INF, 0.0, LOW, LOW]), 2),
                        (torch.tensor([-INF, -INF, -INF, 0.0, LOW, LOW, LOW, LOW]), 4)):
        _, e = chosen(dev, x, 1, "sigmoid", bias, 4, 1, "top2")
        assert e[:, 0].tolist() == [first] * 3, bias
