"""The join's gradient for plans that were changed by hand: a slot taken out of ``position`` has no part in the
join, and its row's gradient is zero (not what the memory held)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,k,N", [(5, 2, 3), (300, 4, 64), (70, 3, 1000)])
def test_slots_taken_out_of_a_plan(dev, T, k, N, dt):
    from nerfhip import experts
    g = torch.Generator().manual_seed(T)
    E = 4
    e = torch.randint(-1, E, (T, k), generator=g, dtype=torch.int32)
    p = experts.plan(e.to(dev), E)
    position = p.position.clone()
    position[torch.rand(T, k, generator=g).to(dev) < 0.4] = -1       # (over a capacity, say)
    p = p._replace(position=position)
    y = torch.randn(T * k, N, generator=g).to(dt)
    w = torch.randn(T, k, generator=g)
    dout = torch.randn(T, N, generator=g).to(dt)
    yl, wl = y.to(dev).requires_grad_(), w.to(dev).requires_grad_()
    out = experts.combine(yl, wl, p)
    junk = torch.full((T * k, N), 7.0, device=dev, dtype=dt)         # what a fresh allocation may find
    del junk
    dy, dw = torch.autograd.grad(out, [yl, wl], dout.to(dev))
    y64, w64 = y.double().requires_grad_(), w.double().requires_grad_()
    pos = position.cpu().long()
    rows = torch.where((pos >= 0)[..., None], y64[pos.clamp_min(0)], torch.zeros((), dtype=torch.float64))
    want = (w64[..., None] * rows).sum(1)
    rdy, rdw = torch.autograd.grad(want, [y64, w64], dout.double())
    half = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}[dt]
    assert bool(((dy.cpu().double() - rdy).abs() <= (2.0 ** -24 + half) * rdy.abs()).all())
    size = (rows.detach() * dout.double()[:, None]).abs().sum(-1)
    assert bool(((dw.cpu().double() - rdw).abs() <= (N + 8) * 2.0 ** -23 * size).all())
    size = (w.double()[..., None] * rows.detach()).abs().sum(1)
    assert bool(((out.detach().cpu().double() - want.detach()).abs() <= (k + 1) * 2.0 ** -23 * size +
                 half * want.detach().abs()).all())
