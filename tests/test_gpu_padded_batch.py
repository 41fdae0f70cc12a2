"""A training batch with padded rows and dropped choices: no part in the join, no gradient from it, and the rest as
64 bits on the CPU have it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,N", [(1, 4, 2, 8), (50, 6, 2, 33), (400, 40, 5, 128)])
def test_padded_rows_and_dropped_choices(T, E, k, N, score):
    from nerfhip import experts
    dev = torch.device("cuda:0")
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, E, generator=g)
    y = torch.randn(T * k, N, generator=g)
    dout = torch.randn(T, N, generator=g)
    drop = torch.rand(T, k, generator=g) < 0.2
    drop[T // 2:] |= torch.rand(T - T // 2, 1, generator=g) < 0.5        # whole rows
    x[T // 2, 0] = float("-inf")
    xl, yl = x.to(dev).requires_grad_(), y.to(dev).requires_grad_()
    w, e = experts.route(xl, k, score=score)
    p = experts.plan(torch.where(drop.to(dev), -1, e), E)
    out = experts.combine(yl, w, p)
    dx, dy = torch.autograd.grad(out, [xl, yl], dout.to(dev))
    x64, y64 = x.double().requires_grad_(), y.double().requires_grad_()
    s = torch.softmax(x64, 1) if score == "softmax" else torch.sigmoid(x64)
    c = torch.gather(s, 1, e.cpu().long())
    c = c / c.sum(1, keepdim=True)
    pos = p.position.cpu().long()
    assert torch.equal(pos < 0, drop)
    rows = torch.where((pos >= 0)[..., None], y64[pos.clamp_min(0)], torch.zeros((), dtype=torch.float64))
    want = (c[..., None] * rows).sum(1)
    rx, ry = torch.autograd.grad(want, [x64, y64], dout.double())
    assert bool((out[drop.all(1).to(dev)] == 0).all()) and bool((dx[drop.all(1).to(dev)] == 0).all())
    # k products of weights within 7e-6 (the gate's own bound), added in 32 bits
    size = (c[..., None] * rows).abs().sum(1).detach()
    assert bool(((out.cpu().double() - want).abs() <= 1e-5 * size).all())
    assert bool(((dy.cpu().double() - ry).abs() <= 1e-5 * ry.abs() + 1e-30).all())
    # a row's gradient: products with N-term sums, differences of them
    dw = (rows * dout.double()[:, None]).abs().sum(-1).amax(1, keepdim=True).detach()
    assert bool(((dx.cpu().double() - rx).abs() <= (N * 2.0 ** -23 + 3e-5) * dw).all())
