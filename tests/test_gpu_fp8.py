"""8-bit block-scaled products (nerfhip/fp8.py, experts.expert_linear) against 64-bit products of the
same 8-bit values on the CPU.

Rounding to blocks is exact arithmetic but for the one rounding to e4m3, so the plain form's 8-bit values are
the kernels'. Sums: K products in float32, any order: (K + 2) 2^-24 of the sum of magnitudes; then half a step
of the output's type. 16-bit results come from the 8-bit matrix instruction, which brings 8 neighbouring products
to the largest one's scale with 13 bits below it: each of the other 7 is off by at most 2^-13 of the largest, so
the sum by at most 7 * 2^-13 of the sum of magnitudes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


def block_scale(top):
    """The least e in [-127, 127] with top <= 448 * 2^e."""
    m, e = torch.frexp(top.double())
    s = e - 9 + (m > 0.875)
    return torch.where(top > 0, s, torch.full_like(s, -127)).clamp(-127, 127)


def rows8(x):
    """What rows of x stand for in blocks of 1 x 128 (64 bits)."""
    M, K = x.shape
    v = torch.zeros(M, -(-K // 128) * 128, dtype=torch.float64)
    v[:, :K] = x.double()
    v = v.view(M, -1, 128)
    s = block_scale(v.abs().amax(-1, keepdim=True))
    q = torch.ldexp(v, -s).float().to(torch.float8_e4m3fn).double()
    return torch.ldexp(q, s).view(M, -1)[:, :K]


def make_weight(dev, *shape, seed=0, dt=torch.float32):
    from nerfhip import fp8
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(*shape, generator=g) * shape[-1] ** -0.5).to(dt)
    return w, fp8.quantize_weight(w.to(dev))


def check(got, xq, wq, bias, relu, dt):
    want = xq @ wq.t()
    size = xq.abs() @ wq.abs().t()
    if bias is not None:
        want = want + bias.double()
        size = size + bias.double().abs()
    if relu:
        want = want.clamp_min(0)
    err = (got.cpu().double() - want).abs()
    own = 0.0 if dt == torch.float32 else 7 * 2.0 ** -13
    tol = ((xq.shape[1] + 2) * 2.0 ** -24 + own) * size + HALF_STEP[dt] * want.abs() + (2.0 ** -25 if dt == torch.float16 else 0)
    assert bool((err <= tol).all()), float((err / tol.clamp_min(1e-300)).max())


@pytest.mark.parametrize("E,N,K", [(None, 1, 1), (None, 130, 100), (None, 256, 256), (3, 70, 300), (2, 128, 129)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_quantize_weight(dev, E, N, K, dt):
    from nerfhip import fp8
    g = torch.Generator().manual_seed(N)
    shape = (N, K) if E is None else (E, N, K)
    w = torch.randn(*shape, generator=g).to(dt)
    w[..., : N // 2, : K // 2] *= 2.0 ** -9
    pad = torch.zeros(*shape[:-2], N + 2, K + 5, dtype=dt)     # a pitch, an odd start
    pad[..., 1:N + 1, 3:K + 3] = w
    wide = pad.to(dev)[..., 1:N + 1, 3:K + 3]
    for f in (fp8.quantize_weight(w.to(dev)), fp8.quantize_weight(wide)):
        for e in range(E or 1):
            v = torch.zeros(-(-N // 128) * 128, -(-K // 128) * 128, dtype=torch.float64)
            v[:N, :K] = (w if E is None else w[e]).double()
            b = v.view(v.shape[0] // 128, 128, -1, 128)
            s = block_scale(b.abs().amax((1, 3), keepdim=True))
            q = torch.ldexp(torch.ldexp(b, -s).float().to(torch.float8_e4m3fn).double(), s).reshape(v.shape)
            got, sc = f.dequantize().cpu().double(), f.scale.cpu().int()
            assert torch.equal(got if E is None else got[e], q[:N, :K])
            assert torch.equal(sc if E is None else sc[e], (s[:, 0, :, 0] + 127).int())
            assert bool((f.q.view(torch.uint8)[..., K:] == 0).all())


SHAPES = [(1, 1, 1), (1, 64, 128), (3, 17, 130), (16, 40, 1000), (17, 33, 64), (16, 4096, 4096), (129, 200, 257),
          (777, 1000, 1111), (300, 128, 2048), (1, 1000, 8192), (4097, 256, 256), (130, 130, 20000)]
LARGE = [(65537, 100, 260, torch.bfloat16), (65536, 256, 256, torch.float16), (65600, 300, 130, torch.float32),
         (70000, 40, 500, torch.bfloat16), (4100, 8200, 4224, torch.bfloat16), (3, 5, 66000, torch.float32),
         (140, 150, 66000, torch.bfloat16)]


@pytest.mark.parametrize("M,N,K,dt", [(*s, dt) for s in SHAPES for dt in (torch.bfloat16, torch.float32, torch.float16)
                                      if dt == torch.bfloat16 or s[0] * s[1] * s[2] <= 1 << 28])
def test_linear(dev, M, N, K, dt):
    from nerfhip import fp8
    g = torch.Generator().manual_seed(M + N + K)
    w, f = make_weight(dev, N, K, seed=K)
    x = (torch.randn(M, K, generator=g) * torch.exp(torch.randn(1, K, generator=g))).to(dt)
    bias = torch.randn(N, generator=g)
    wq, xq = f.dequantize().cpu().double(), rows8(x)
    check(fp8.linear(x.to(dev), f), xq, wq, None, False, dt)
    check(fp8.linear(x.to(dev), f, bias=bias.to(dev), relu=True, out_dtype=torch.float32), xq, wq, bias, True,
          torch.float32)
    # rows with a pitch and an odd start
    wide = torch.zeros(M, K + 3, dtype=dt)
    wide[:, 1:K + 1] = x
    assert torch.equal(fp8.linear(wide.to(dev)[:, 1:K + 1], f), fp8.linear(x.to(dev), f))


@pytest.mark.parametrize("M,N,K,dt", LARGE)
def test_linear_large(dev, M, N, K, dt):
    """The forms for many short rows, long rows with many tiles, and more blocks than scales fit into LDS:
    rows from all over, against 64 bits."""
    from nerfhip import fp8
    g = torch.Generator(device="cuda").manual_seed(M)
    f = fp8.quantize_weight(torch.randn(N, K, device=dev, generator=g) * K ** -0.5)
    x = torch.randn(M, K, device=dev, generator=g).to(dt)
    bias = torch.randn(N, device=dev, generator=g)
    y = fp8.linear(x, f, bias=bias)
    rows = torch.unique(torch.cat([torch.arange(0, M, max(1, M // 150)), torch.arange(max(0, M - 130), M)]))
    check(y[rows.to(dev)], rows8(x[rows.to(dev)].cpu()), f.dequantize().cpu().double(), bias.cpu(), False, dt)
    assert bool(torch.isfinite(y).all())


def test_linear_takes_any_leading_axes_and_layouts(dev):
    from nerfhip import fp8
    _, f = make_weight(dev, 24, 96)
    x = torch.randn(2, 3, 5, 96, device=dev)
    y = fp8.linear(x, f)
    assert y.shape == (2, 3, 5, 24)
    assert torch.equal(y, fp8.linear(x.reshape(-1, 96), f).view_as(y))
    xt = torch.randn(96, 40, device=dev)
    assert torch.equal(fp8.linear(xt.t(), f), fp8.linear(xt.t().contiguous(), f))
    one = torch.randn(1, 96, device=dev)
    assert torch.equal(fp8.linear(one.expand(40, 96), f), fp8.linear(one.repeat(40, 1), f))
    assert fp8.linear(torch.empty(0, 96, device=dev), f).shape == (0, 24)
    assert fp8.linear(torch.randn(96, device=dev), f).shape == (24,)


@pytest.mark.parametrize("M", [2, 40])
def test_extreme_and_non_finite_values(dev, M):
    """Scales from 2^-127 to the largest, zeros, and rows with NaN or infinity (NaN outputs, other rows
    untouched)."""
    from nerfhip import fp8
    w, f = make_weight(dev, 40, 256)
    g = torch.Generator().manual_seed(9)
    x = torch.randn(M, 256, generator=g)
    x[0, :128] = 0.0
    x[0, 128:] *= 2.0 ** -60
    xs = x.clone()
    wq = f.dequantize().cpu().double()
    check(fp8.linear(x.to(dev), f), rows8(x), wq, None, False, torch.float32)
    xs[1, 7] = 3e38
    xs[1, 200] = 1e-44
    big = fp8.linear(xs.to(dev) * 2.0 ** -20, f)
    check(big, rows8(xs * 2.0 ** -20), wq, None, False, torch.float32)
    for v in (math.nan, math.inf, -math.inf):
        xs = x.clone()
        xs[1, 200] = v
        y = fp8.linear(xs.to(dev), f, relu=True)
        assert bool(torch.isnan(y[1]).all())
        keep = [i for i in range(M) if i != 1]
        assert torch.equal(y[keep], fp8.linear(x.to(dev), f, relu=True)[keep])
    bad = w.clone()
    bad[3, 5] = math.inf
    y = fp8.linear(x.to(dev), fp8.quantize_weight(bad.to(dev)))
    assert bool(torch.isnan(y).all())        # (the block's 128 rows of weights share its scale)


@pytest.mark.parametrize("T,k,E,N,K", [(1, 1, 1, 16, 16), (1, 4, 8, 100, 200), (16, 6, 64, 96, 256), (40, 2, 3, 130, 129),
                                       (600, 3, 5, 200, 384), (64, 1, 300, 16, 128), (257, 2, 2, 128, 1000),
                                       (16500, 4, 7, 130, 200)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_expert_linear(dev, T, k, E, N, K, dt):
    from nerfhip import experts
    g = torch.Generator().manual_seed(T + E)
    w, f = make_weight(dev, E, N, K, seed=E)
    x = torch.randn(T, K, generator=g).to(dt)
    e = (torch.rand(T, k, generator=g) ** 3 * E).int().clamp_max(E - 1)    # some experts with many rows, some with none
    if T > 4:
        e[1] = -1
        e[T // 2, 0] = E + 7
    p = experts.plan(e.to(dev), E)
    bias = torch.randn(E, N, generator=g)
    y = experts.expert_linear(x.to(dev), f, p, gather=True, bias=bias.to(dev), relu=True)
    xq, wq = rows8(x), f.dequantize().cpu().double()
    off, order = p.offsets.cpu().tolist(), p.order.cpu().long()
    for i in range(E):
        if off[i + 1] > off[i]:
            check(y[off[i]:off[i + 1]], xq[order[off[i]:off[i + 1]] // k], wq[i], bias[i], True, dt)
    assert bool((y[off[E]:] == 0).all())
    rows = x.to(dev)[(p.order.clamp_min(0) // k).long()]
    assert torch.equal(experts.expert_linear(rows, f, p, bias=bias.to(dev), relu=True), y)


@pytest.mark.parametrize("n", [24, 700])
def test_rows_that_a_plan_leaves_out(dev, n):
    """A plan made by hand: sorted rows whose slot is no row of x count as rows of zeros (bias alone), in the
    skinny and the tiled form; sorted rows behind the last expert's become zeros."""
    from nerfhip import experts
    E, N, K = 2, 40, 200
    _, f = make_weight(dev, E, N, K)
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, K, generator=g)
    bias = torch.randn(E, N, generator=g)
    order = torch.randperm(n, generator=g).int()
    order[::3] = -1
    order[1] = 2 ** 31 - 1
    order[2] = n
    off = torch.tensor([0, n // 2, n - 5], dtype=torch.int32)
    p = experts.Plan(order.to(dev), torch.zeros(n, 1, dtype=torch.int32, device=dev), off.to(dev))
    y = experts.expert_linear(x.to(dev), f, p, gather=True, bias=bias.to(dev)).cpu()
    xq, wq = rows8(x), f.dequantize().cpu().double()
    for e in range(E):
        rows = torch.arange(int(off[e]), int(off[e + 1]))
        src = order[rows].long()
        live = (src >= 0) & (src < n)
        assert bool((y[rows[~live]] == bias[e]).all())
        check(y[rows[live]], xq[src[live]], wq[e], bias[e], False, torch.float32)
    assert bool((y[n - 5:] == 0).all())


def test_served_experts_end_to_end(dev):
    """Gate, plan, two 8-bit layers and the join, for a batch and for a single row (which takes the
    skinny form): row by row against the 64-bit form with the same roundings between the layers."""
    from nerfhip import experts
    g = torch.Generator().manual_seed(2)
    T, E, k, D, H = 70, 4, 2, 128, 256
    _, f1 = make_weight(dev, E, H, D, seed=1)
    _, f2 = make_weight(dev, E, D, H, seed=2)
    x = torch.randn(T, D, generator=g).to(torch.bfloat16)
    logits = torch.randn(T, E, generator=g)

    def layer(x, logits):
        w, e = experts.route(logits, k)
        p = experts.plan(e, E)
        h = experts.expert_linear(x, f1, p, gather=True, relu=True)
        return experts.combine(experts.expert_linear(h, f2, p, out_dtype=torch.float32), w, p), w, e, h, p

    out, w, e, h, p = layer(x.to(dev), logits.to(dev))
    one = torch.cat([layer(x[i:i + 1].to(dev), logits[i:i + 1].to(dev))[0] for i in range(8)])
    w1, w2 = f1.dequantize().cpu().double(), f2.dequantize().cpu().double()
    xq, hq = rows8(x), rows8(h.cpu())
    pos, want = p.position.cpu(), torch.zeros(T, D, dtype=torch.float64)
    for t in range(T):
        for j in range(k):
            i, r = int(e[t, j]), int(pos[t, j])
            first = (w1[i] @ xq[t]).clamp_min(0)
            assert float((h[r].cpu().double() - first).abs().max()) <= 2.0 ** -8 * float(first.max()) + 1e-4
            want[t] += float(w[t, j]) * (w2[i] @ hq[r])
    assert float((out.cpu().double() - want).abs().max()) < 1e-4 * float(want.abs().max())
    # single rows: the hidden layer's sums may round to 16 bits the other way, so 8-bit steps may differ
    assert float((one - out[:8]).norm() / out[:8].norm()) < 0.01


def test_calls_on_another_stream_and_in_a_graph(dev):
    from nerfhip import experts, fp8
    _, f = make_weight(dev, 200, 300)
    _, fe = make_weight(dev, 4, 64, 300)
    xs = [torch.randn(90, 300, device=dev) for _ in range(3)]
    lg = [torch.randn(90, 4, device=dev) for _ in range(3)]

    def step(x, l):
        w, e = experts.route(l, 2, score="sigmoid", bias=torch.zeros(4, device=dev))
        p = experts.plan(e, 4)
        return fp8.linear(x, f), experts.combine(experts.expert_linear(x, fe, p, gather=True), w, p)

    want = [step(x, l) for x, l in zip(xs, lg)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(xs[0], lg[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    x, l = xs[0].clone(), lg[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, l)
    for _ in range(2):
        for i in range(3):
            x.copy_(xs[i])
            l.copy_(lg[i])
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
            step(xs[2], lg[2])       # eager work between the replays


def test_two_streams_at_once(dev):
    """Products of every form on two streams, nothing waiting between: as one after the other."""
    from nerfhip import experts, fp8
    _, f1 = make_weight(dev, 300, 700, seed=1)
    _, f2 = make_weight(dev, 256, 200, seed=2)
    _, fe = make_weight(dev, 8, 96, 260, seed=3)
    xs = [torch.randn(m, 700, device=dev) for m in (1, 20, 500, 1300)]
    ys = [torch.randn(m, 200, device=dev).bfloat16() for m in (7, 40000, 33000, 600)]
    zs = [torch.randn(m, 260, device=dev) for m in (5, 50, 400, 900)]
    plans = [experts.plan(torch.randint(-1, 8, (z.shape[0], 3), device=dev, dtype=torch.int32), 8) for z in zs]

    def first(i):
        return fp8.linear(xs[i], f1), experts.expert_linear(zs[i], fe, plans[i], gather=True)

    def second(i):
        return (fp8.linear(ys[i], f2),)

    want = [(*first(i), *second(i)) for i in range(4)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for i in range(4):
        with torch.cuda.stream(s1):
            a = first(i)
        with torch.cuda.stream(s2):
            b = second(i)
        got.append((*a, *b))
    torch.cuda.synchronize()
    for u, v in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(u, v))
