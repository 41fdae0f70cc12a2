"""Muon where |g| is far below eps: X = g / (|g| + eps) is tiny then, and so is the result.

Bound, relative to the result's norm: a step's own error is the 2^-19 of |X| of test_gpu_muon.py, and what is there
already grows by p's slope, 3.4445 while the singular values (t 3.4445^k at most, t = |g| / (|g| + eps)) are below
1.1, 4 beyond. While they are small |X| itself grows by 3.4445, so relative errors add up and do not grow: steps + 1
times 2^-19."""
import math

import pytest
import torch

from test_gpu_muon import A, B, C, HALF_STEP

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


def ref(g, steps=5, eps=1e-7):
    """(NS(g), the bound of its error's norm)."""
    x = g.double()
    if x.shape[0] > x.shape[1]:
        y, err = ref(g.t(), steps, eps)
        return y.t(), err
    t = float(x.norm() / (x.norm() + eps))
    x = x / (x.norm() + eps)
    err = 2.0 ** -19 * float(x.norm())
    for k in range(steps):
        a = x @ x.t()
        y = A * x + (B * a + C * (a @ a)) @ x
        err = (A if t * A ** k < 1.1 else 4.0) * err + 2.0 ** -19 * max(float(x.norm()), float(y.norm()))
        x = y
    return x, err


def check(got, g, steps=5, eps=1e-7):
    want, tol = ref(g, steps, eps)
    if got.dtype != torch.float32:
        tol += HALF_STEP[got.dtype] * float(want.norm())
    if got.dtype == torch.float16:
        tol += 2.0 ** -25 * math.sqrt(want.numel())
    err = float((got.cpu().double() - want).norm())
    assert err <= tol, (err, tol, float(want.norm()))


@pytest.mark.parametrize("size", [1e-8, 1e-9, 1e-10, 1e-12, 1e-16, 1e-25, 1e-33])
@pytest.mark.parametrize("m,n", [(16, 16), (256, 256), (300, 70), (40, 1000)])
def test_matrices_far_below_eps(dev, size, m, n):
    from nerfhip import muon
    g = torch.randn(m, n, generator=torch.Generator().manual_seed(m))
    g = g / g.norm() * size
    for steps in (1, 5, 12):
        check(muon.orthogonalize(g.to(dev), steps=steps), g, steps)


def test_a_stack_of_all_sizes(dev):
    """Each matrix has its own scale, through the large tiles and the small ones."""
    from nerfhip import muon
    size = torch.tensor([1.0, 1e-6, 1e-7, 1e-8, 1e-11, 0.0, 1e-20, 1e10])
    for m, n in ((64, 96), (700, 900)):
        g = torch.randn(8, m, n, generator=torch.Generator().manual_seed(3))
        g = g / g.flatten(1).norm(dim=1)[:, None, None] * size[:, None, None]
        for v in (g, g.transpose(1, 2).contiguous()):
            out = muon.orthogonalize(v.to(dev))
            for i in range(8):
                check(out[i], v[i])


@pytest.mark.parametrize("eps", [1e-3, 1e-30, 1e-44, 1e30])
def test_eps_of_all_sizes(dev, eps):
    """Zeros stay zeros, whatever eps that is a positive 32-bit number."""
    from nerfhip import muon
    g = torch.randn(3, 40, 50, generator=torch.Generator().manual_seed(4))
    g[1] = 0.0
    out = muon.orthogonalize(g.to(dev), eps=eps)
    assert torch.equal(out[1].cpu(), torch.zeros_like(g[1]))
    e32 = float(torch.tensor(eps, dtype=torch.float32))
    for i in (0, 2):
        check(out[i], g[i], eps=e32)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_16_bit_gradients_far_below_eps(dev, dt):
    from nerfhip import muon
    g = (torch.randn(64, 80, generator=torch.Generator().manual_seed(5)) * 1e-6).to(dt)
    check(muon.orthogonalize(g.to(dev), eps=1e-2), g, eps=float(torch.tensor(1e-2)))


def test_not_finite_beside_tiny(dev):
    from nerfhip import muon
    g = torch.randn(3, 70, 90, generator=torch.Generator().manual_seed(2)) * 1e-15
    g[1, 3, 3] = math.nan
    g[2, 3, 3] = math.inf
    out = muon.orthogonalize(g.to(dev))
    check(out[0], g[0])
    assert bool(torch.isnan(out[1:]).all())


def test_an_update_by_a_tiny_gradient(dev):
    """The step is -lr sqrt(max(1, m / n)) X all the same."""
    from nerfhip import muon
    g = torch.randn(64, 32, generator=torch.Generator().manual_seed(6)) * 1e-13
    p, b = torch.zeros(64, 32, device=dev), torch.zeros(64, 32, device=dev)
    muon.muon_update([p], [g.to(dev)], [b], 1.0)
    check(p * -(2.0 ** -0.5), g.double() * 1.95)
