"""More rows than one launch of the gate takes: every row is chosen for, and every row has its gradient."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,E", [((1 << 26) + 37, 2), ((1 << 28) + 37, 2), ((1 << 24) + 5, 300)])
def test_rows_of_several_launches(T, E):
    from nerfhip import experts
    dev = torch.device("cuda:0")
    if torch.cuda.mem_get_info()[0] < 48 << 30:
        pytest.skip("needs 48 GB")
    x = torch.empty(T, E, device=dev, dtype=torch.float16)
    x.normal_(generator=torch.Generator(device=dev).manual_seed(1))
    x.requires_grad_()
    w, e = experts.route(x, 1, renormalise=False)
    (d,) = torch.autograd.grad(w, x, torch.ones_like(w))
    for t in range(0, T, 1 << 24):
        v = x.detach()[t:t + (1 << 24)]
        top, at = v.max(1)
        mine = e[t:t + (1 << 24), 0].long()
        assert torch.equal(v.gather(1, mine[:, None])[:, 0], top)
        assert bool((v.argmax(1) >= mine).all())                       # ties: the lowest index
        p = torch.softmax(v.float(), 1)
        best = p.gather(1, mine[:, None])
        assert float((w.detach()[t:t + (1 << 24)] - best).abs().max()) < 1e-6
        want = -best * p
        want.scatter_add_(1, mine[:, None], best)
        assert float((d[t:t + (1 << 24)].float() - want).abs().max()) < 2.0 ** -11 * 0.25 + 1e-6
