"""The 8-bit product's forms at the sizes and types that test_gpu_fp8.py does not reach: the resident form (32768
rows or more, N and K up to 256) with both of its tiles, one and two blocks of K, narrow matrices, ragged rows, every
type and alignment; experts' rows through 256 x 256 tiles; experts in float16; all rows on one expert. Tolerances are
those of test_gpu_fp8.py."""
import pytest
import torch

from test_gpu_fp8 import check, make_weight, rows8

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


RESIDENT = [(32768, 256, 256, F32, F32), (32769, 100, 130, F32, F32), (40001, 256, 64, BF16, BF16),
            (33000, 130, 256, BF16, F32), (32799, 1, 1, F32, F16), (32768, 128, 128, F16, BF16),
            (33333, 129, 129, F16, F16), (32831, 255, 255, F32, BF16), (50000, 7, 100, F16, F32),
            (32895, 256, 129, BF16, F16), (65536, 64, 16, F32, F32)]


@pytest.mark.parametrize("M,N,K,dt,out", RESIDENT)
@pytest.mark.parametrize("relu", [False, True])
def test_resident(dev, M, N, K, dt, out, relu):
    from nerfhip import fp8
    g = torch.Generator(device="cuda").manual_seed(M + N)
    w, f = make_weight(dev, N, K, seed=K)
    x = (torch.randn(M, K, device=dev, generator=g) * torch.exp(torch.randn(M, 1, device=dev, generator=g))).to(dt)
    bias = torch.randn(N, device=dev, generator=g) if relu or N > 100 else None
    wide = torch.zeros(M, K + 3, device=dev, dtype=dt)       # a pitch and an odd start
    wide[:, 1:K + 1] = x
    rows = torch.unique(torch.cat([torch.arange(0, M, max(1, M // 300)), torch.arange(M - 200, M)]))
    xq, wq = rows8(x[rows.to(dev)].cpu()), f.dequantize().cpu().double()
    y = fp8.linear(x, f, bias=bias, relu=relu, out_dtype=out)
    assert y.dtype == out and y.shape == (M, N)
    check(y[rows.to(dev)], xq, wq, None if bias is None else bias.cpu(), relu, out)
    assert torch.equal(fp8.linear(wide[:, 1:K + 1], f, bias=bias, relu=relu, out_dtype=out), y)
    # every row: the same rows in calls too short for this form, whose sums may be in another order
    part = torch.cat([fp8.linear(v, f, bias=bias, relu=relu, out_dtype=out) for v in x.split(16000)])
    size = float(y.double().abs().max())
    assert float((part.double() - y.double()).abs().max()) <= (2.0 ** -7 if out != F32 else 2.0 ** -16) * size


def test_resident_rows_that_are_not_finite(dev):
    from nerfhip import fp8
    _, f = make_weight(dev, 200, 200)
    x = torch.randn(33000, 200, device=dev)
    want = fp8.linear(x, f, relu=True)
    x[17, 3], x[32999, 199], x[20000, 0] = float("nan"), float("inf"), -float("inf")
    y = fp8.linear(x, f, relu=True)
    bad = torch.zeros(33000, dtype=torch.bool, device=dev)
    bad[[17, 32999, 20000]] = True
    assert bool(torch.isnan(y[bad]).all()) and torch.equal(y[~bad], want[~bad])


def check_experts(dev, x, f, p, k, y, bias, relu, out, every=1):
    off, order, wq = p.offsets.cpu().tolist(), p.order.cpu().long(), f.dequantize().cpu().double()
    for i in range(len(off) - 1):
        rows = torch.arange(off[i], off[i + 1])[::every]
        if len(rows):
            check(y[rows.to(dev)], rows8(x[order[rows] // k]), wq[i], None if bias is None else bias[i], relu, out)
    assert bool((y[off[-1]:] == 0).all())


@pytest.mark.parametrize("dt,out", [(BF16, BF16), (F16, F16), (F32, BF16)])
def test_experts_through_the_largest_tiles(dev, dt, out):
    """K of 4096 and more, 512 tiles of 256 x 256 and more."""
    from nerfhip import experts
    g = torch.Generator().manual_seed(7)
    T, k, E, N, K = 4100, 2, 3, 4200, 4100
    _, f = make_weight(dev, E, N, K, seed=E)
    x = torch.randn(T, K, generator=g).to(dt)
    e = (torch.rand(T, k, generator=g) ** 2 * E).int().clamp_max(E - 1)
    e[5] = -1
    p = experts.plan(e.to(dev), E)
    bias = torch.randn(E, N, generator=g)
    y = experts.expert_linear(x.to(dev), f, p, gather=True, bias=bias.to(dev), relu=True, out_dtype=out)
    check_experts(dev, x, f, p, k, y, bias, True, out, every=97)
    rows = x.to(dev)[(p.order.clamp_min(0) // k).long()]
    assert torch.equal(experts.expert_linear(rows, f, p, bias=bias.to(dev), relu=True, out_dtype=out), y)


@pytest.mark.parametrize("T,k,E,N,K", [(1, 1, 1, 16, 16), (16, 6, 64, 96, 256), (40, 2, 3, 130, 129), (600, 3, 5, 200, 384)])
@pytest.mark.parametrize("out", [F16, F32])
def test_experts_in_float16(dev, T, k, E, N, K, out):
    from nerfhip import experts
    g = torch.Generator().manual_seed(T + E)
    _, f = make_weight(dev, E, N, K, seed=E)
    x = torch.randn(T, K, generator=g).half()
    p = experts.plan(torch.randint(-1, E, (T, k), generator=g, dtype=torch.int32).to(dev), E)
    y = experts.expert_linear(x.to(dev), f, p, gather=True, out_dtype=out)
    check_experts(dev, x, f, p, k, y, None, False, out)


@pytest.mark.parametrize("T,E,N,K", [(1024, 64, 200, 300), (1000, 64, 64, 128), (17, 2, 40, 256), (33, 3, 130, 129),
                                     (4096, 300, 48, 200), (1, 5, 16, 16)])
@pytest.mark.parametrize("kind", ["one", "last", "two", "none", "most dropped"])
@pytest.mark.parametrize("out", [BF16, F32])
def test_uneven_experts(dev, T, E, N, K, kind, out):
    """Up to 16 rows an expert on average, all of them on one expert, on two, on none."""
    from nerfhip import experts
    g = torch.Generator().manual_seed(T + E)
    _, f = make_weight(dev, E, N, K, seed=E)
    x = torch.randn(T, K, generator=g).bfloat16()
    e = torch.full((T, 1), {"one": E // 2, "last": E - 1, "two": 0, "none": -1, "most dropped": E}[kind], dtype=torch.int32)
    if kind == "two":
        e[::2] = E - 1
    elif kind == "most dropped":
        e[::5] = torch.randint(0, E, (len(e[::5]), 1), generator=g, dtype=torch.int32)
    p = experts.plan(e.to(dev), E)
    bias = torch.randn(E, N, generator=g)
    y = torch.full((T, N), 3.0, device=dev, dtype=out)       # what a fresh allocation may find
    del y
    y = experts.expert_linear(x.to(dev), f, p, gather=True, bias=bias.to(dev), relu=True, out_dtype=out)
    check_experts(dev, x, f, p, 1, y, bias, True, out)
    assert torch.equal(y, experts.expert_linear(x.to(dev)[p.order.clamp_min(0).long()], f, p, bias=bias.to(dev), relu=True,
                                                out_dtype=out))
