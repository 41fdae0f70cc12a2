"""Gated experts (nerfhip/experts.py on csrc/experts_ops.hip) against plain 64-bit forms on the CPU.

Choices, plans and offsets have to be equal. Weights: the exponentials (1 ulp each), one division and at
most k additions in float32 stay below 16 steps of 2^-24 relative (1e-6); a logit difference d under exp
adds |d| 2^-24, at most 100 of them here (6e-6). Joins: k products and additions in float32 of |w y|, then half
a step of the output's type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -9 * 2, torch.float16: 2.0 ** -12 * 2}


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


def ref_scores(x, score):
    x = x.double()
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-x))
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    return e / e.sum(1, keepdim=True)


def ref_choice(x, k, score, bias, groups, top_groups, group_score):
    T, E = x.shape
    low = torch.finfo(torch.float64).min
    s = ref_scores(x, score)
    key = x.double() if bias is None else s + bias.double()
    key = torch.where(key > low, key, torch.full_like(key, low))       # NaN and -inf: the lowest number
    if groups > 1:
        base = key if bias is not None or group_score == "max" else s
        best = torch.sort(base.view(T, groups, -1), -1, descending=True)[0]
        g = best[..., :2].sum(-1) if group_score == "top2" else best[..., 0]
        order = torch.sort(g, dim=1, descending=True, stable=True)[1][:, :top_groups]
        keep = torch.zeros_like(g, dtype=torch.bool).scatter_(1, order, True).repeat_interleave(E // groups, 1)
        key = torch.where(keep, key, torch.full_like(key, -math.inf))
    return torch.sort(key, dim=1, descending=True, stable=True)[1][:, :k]


def ref_weights(x, experts, score, renorm, scale):
    s = ref_scores(x, score)
    c = torch.gather(s, 1, experts)
    return scale * (c / c.sum(1, keepdim=True) if renorm else c)


CASES = [  # T, E, k, score, bias, groups, top_groups, group_score, renorm, dtype
    (1, 1, 1, "softmax", False, 1, 1, "max", True, torch.float32),
    (1, 64, 6, "softmax", False, 1, 1, "max", True, torch.float32),
    (17, 5, 5, "sigmoid", True, 1, 1, "max", True, torch.float32),
    (33, 7, 3, "softmax", True, 1, 1, "max", False, torch.bfloat16),
    (100, 64, 2, "softmax", False, 1, 1, "max", False, torch.float16),
    (257, 100, 8, "sigmoid", True, 4, 2, "top2", True, torch.bfloat16),
    (301, 128, 4, "softmax", True, 8, 3, "max", True, torch.float32),
    (1021, 256, 8, "sigmoid", True, 8, 4, "top2", True, torch.bfloat16),
    (130, 258, 32, "softmax", False, 3, 2, "top2", True, torch.float16),
    (70, 512, 16, "sigmoid", False, 16, 5, "top2", False, torch.float32),
    (65, 1024, 8, "softmax", True, 64, 7, "top2", True, torch.float32),
    (66, 1000, 9, "sigmoid", False, 4, 1, "max", True, torch.bfloat16),
    (5000, 12, 2, "softmax", True, 6, 6, "top2", True, torch.float32),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"T{c[0]}-E{c[1]}-k{c[2]}-{c[3]}-g{c[5]}")
def test_route_matches_the_exact_choice(dev, case):
    from nerfhip import experts
    T, E, k, score, with_bias, groups, top, gs, renorm, dt = case
    g = torch.Generator().manual_seed(T + E)
    x = (2.0 * torch.randn(T, E, generator=g)).to(dt)
    bias = 0.1 * torch.randn(E, generator=g) if with_bias else None
    w, e = experts.route(x.to(dev), k, score=score, bias=None if bias is None else bias.to(dev), groups=groups,
                         top_groups=top, group_score=gs, renormalise=renorm, scale=1.5)
    want = ref_choice(x, k, score, bias, groups, top, gs)
    assert torch.equal(e.cpu().long(), want)
    rw = ref_weights(x, want, score, renorm, 1.5)
    assert float(((w.cpu().double() - rw) / rw).abs().max()) < 7e-6
    # a row pitch and an odd start
    wide = torch.zeros(T, E + 3, dtype=dt)
    wide[:, 1:E + 1] = x
    w2, e2 = experts.route(wide.to(dev)[:, 1:E + 1], k, score=score, bias=None if bias is None else bias.to(dev),
                           groups=groups, top_groups=top, group_score=gs, renormalise=renorm, scale=1.5)
    assert torch.equal(e, e2) and torch.equal(w, w2)


def test_keys_nearer_than_float32_are_told_apart(dev):
    """Biases that bring pairs of experts' keys to within 1e-9 of each other, either way round."""
    from nerfhip import experts
    g = torch.Generator().manual_seed(3)
    T, E = 512, 32
    for score in ("sigmoid", "softmax"):
        x = torch.randn(1, E, generator=g).repeat(T, 1)
        s = ref_scores(x[:1], score)[0]
        bias = (2.0 - s).float()                       # every key within float32's steps of 2
        x = x + 1e-6 * torch.randn(T, E, generator=g)  # .. and each row another order
        want = ref_choice(x, 8, score, bias, 1, 1, "max")
        _, e = experts.route(x.to(dev), 8, score=score, bias=bias.to(dev))
        assert torch.equal(e.cpu().long(), want), score
        want = ref_choice(x, 8, score, bias, 8, 3, "top2")
        _, e = experts.route(x.to(dev), 8, score=score, bias=bias.to(dev), groups=8, top_groups=3, group_score="top2")
        assert torch.equal(e.cpu().long(), want), score


def test_ties_go_to_the_lowest_index(dev):
    from nerfhip import experts
    x = torch.zeros(3, 64)
    x[1, 40:44] = 1.0
    x[2, ::2] = -0.0
    for bias in (None, torch.zeros(64)):
        _, e = experts.route(x.to(dev), 6, bias=None if bias is None else bias.to(dev))
        assert e.cpu().tolist() == [[0, 1, 2, 3, 4, 5], [40, 41, 42, 43, 0, 1], [0, 1, 2, 3, 4, 5]]
    _, e = experts.route(x.to(dev), 2, groups=8, top_groups=1, group_score="top2")
    assert e.cpu().tolist() == [[0, 1], [40, 41], [0, 1]]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("biased", [True, False])
def test_masked_and_non_finite_logits(dev, score, renorm, biased):
    from nerfhip import experts
    inf, nan = math.inf, math.nan
    low = torch.finfo(torch.float32).min
    x = torch.randn(8, 20, generator=torch.Generator().manual_seed(1))
    x[0] = -inf                     # nothing is left
    x[1, 3:] = -inf                 # fewer than k are left
    x[2, 5] = nan
    x[3] = low                      # masks of the type's lowest value
    x[4, :18] = low
    x[5] = -200.0 + x[5]            # scores below float32's range
    x[6, 7] = inf
    x[7] = nan
    bias = torch.zeros(20).to(dev) if biased else None
    w, e = experts.route(x.to(dev), 5, score=score, bias=bias, renormalise=renorm)
    w, e = w.cpu(), e.cpu().long()
    for r in range(8):
        assert len(set(e[r].tolist())) == 5 and 0 <= int(e[r].min()) and int(e[r].max()) < 20
    assert torch.equal(w[0], torch.zeros(5))
    assert set(e[1, :3].tolist()) == {0, 1, 2} and torch.equal(w[1, 3:], torch.zeros(2))
    assert torch.isnan(w[2]).all() and torch.isnan(w[7]).all()
    if not (biased and score == "softmax"):
        assert 5 not in e[2].tolist()   # (softmax of a row with NaN has no keys but NaN)
    assert torch.isfinite(w[3:6]).all()
    if renorm:
        assert torch.allclose(w[4, :2].sum(), torch.ones(())) and torch.equal(w[4, 2:], torch.zeros(3))
        r5 = x[5].double().gather(0, e[5])
        r5 = torch.exp(r5 - r5.max())       # far below zero sigmoid is exp
        assert float((w[5].double() - r5 / r5.sum()).abs().max()) < 1e-6
    assert torch.isnan(w[6]).all() if score == "softmax" else torch.isfinite(w[6]).all()


def test_a_bias_of_minus_infinity_forbids_an_expert(dev):
    from nerfhip import experts
    x = torch.randn(300, 33, generator=torch.Generator().manual_seed(1))
    bias = torch.zeros(33)
    bias[::2] = -math.inf
    _, e = experts.route(x.to(dev), 16, score="sigmoid", bias=bias.to(dev))
    assert bool((e % 2 == 1).all())
    w, e = experts.route(x.to(dev), 17, score="sigmoid", bias=bias.to(dev))   # one more than are allowed
    assert bool((e[:, :16] % 2 == 1).all()) and bool((e[:, 16] == 0).all()) and bool(torch.isfinite(w).all())


GRADS = [(37, 9, 3, "softmax", True), (37, 9, 3, "softmax", False), (50, 70, 4, "sigmoid", True),
         (50, 70, 4, "sigmoid", False), (20, 260, 8, "softmax", True), (20, 600, 32, "sigmoid", True),
         (3, 1024, 2, "softmax", False), (9, 64, 1, "softmax", True)]


@pytest.mark.parametrize("T,E,k,score,renorm", GRADS)
def test_route_gradient(dev, T, E, k, score, renorm):
    """Against the formula's gradient in 64 bits (errors: some 20 float32 steps of the largest entry) and
    against central differences of the plain form."""
    from nerfhip import experts
    g = torch.Generator().manual_seed(E)
    x = torch.randn(T, E, generator=g)
    dw = torch.randn(T, k, generator=g)
    leaf = x.to(dev).requires_grad_()
    w, e = experts.route(leaf, k, score=score, renormalise=renorm, scale=2.5)
    (d,) = torch.autograd.grad(w, leaf, dw.to(dev))
    e = e.cpu().long()

    def f(v):
        return (ref_weights(v, e, score, renorm, 2.5) * dw.double()).sum(1)

    xd = x.double().requires_grad_()
    (want,) = torch.autograd.grad(f(xd).sum(), xd)
    top = float(want.abs().max()) or 1.0
    assert float((d.cpu().double() - want).abs().max()) < 20 * 2.0 ** -23 * max(top, 1.0)
    h = 1e-5
    for c in {0, int(e[0, 0]), E - 1}:
        step = torch.zeros(T, E, dtype=torch.float64)
        step[:, c] = h
        diff = (f(x.double() + step) - f(x.double() - step)) / (2 * h)
        assert float((d.cpu().double()[:, c] - diff).abs().max()) < 1e-5
    for dt in (torch.bfloat16, torch.float16):
        leaf = x.to(dev, dt).requires_grad_()
        w, e2 = experts.route(leaf, k, score=score, renormalise=renorm, scale=2.5)
        (d16,) = torch.autograd.grad(w, leaf, dw.to(dev))
        assert d16.dtype == dt
        xd = leaf.detach().cpu().double().requires_grad_()
        e16 = e2.cpu().long()
        (want,) = torch.autograd.grad((ref_weights(xd, e16, score, renorm, 2.5) * dw.double()).sum(), xd)
        err = (d16.cpu().double() - want).abs() - HALF_STEP[dt] * want.abs()
        # below the type's least normal number the steps are absolute (float16: half of 2^-24)
        assert float(err.max()) < 20 * 2.0 ** -23 * max(float(want.abs().max()), 1.0) + (2.0 ** -25 if dt == torch.float16 else 0)


def test_rows_without_a_choice_have_no_gradient(dev):
    from nerfhip import experts
    x = torch.randn(4, 12)
    x[1] = -math.inf
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            leaf = x.to(dev).requires_grad_()
            w, _ = experts.route(leaf, 3, score=score, renormalise=renorm)
            (d,) = torch.autograd.grad(w.sum() + (w * w).sum(), leaf)
            assert torch.equal(d[1], torch.zeros_like(d[1])) and bool(torch.isfinite(d).all())


def test_no_rows(dev):
    from nerfhip import experts
    w, e = experts.route(torch.empty(0, 8, device=dev, requires_grad=True), 2)
    p = experts.plan(e, 8)
    assert w.shape == (0, 2) and e.shape == (0, 2) and p.offsets.tolist() == [0] * 9 and p.order.numel() == 0
    out = experts.combine(torch.empty(0, 5, device=dev), w.detach(), p)
    assert out.shape == (0, 5)


# ---------------------------------------------------------------- the plan

@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (1, 6, 64), (7, 3, 5), (1024, 4, 512), (1025, 4, 512), (4096, 1, 1000),
                                   (2048, 2, 1024), (3, 32, 1024), (5000, 2, 16),
                                   (2048, 4, 100), (2731, 3, 200), (8191, 1, 513), (70001, 3, 100), (65536, 8, 256)])
@pytest.mark.parametrize("holes", [False, True])
def test_plan_is_the_stable_sort(dev, T, k, E, holes):
    from nerfhip import experts
    g = torch.Generator().manual_seed(T)
    e = (torch.rand(T, k, generator=g) ** 2 * E).int().clamp_max(E - 1)      # uneven
    if holes:
        e[torch.rand(T, k, generator=g) < 0.3] = -1
        e[torch.rand(T, k, generator=g) < 0.1] = E
        e[0, 0] = 2 ** 31 - 1
    p = experts.plan(e.to(dev), E)
    flat = e.reshape(-1).long()
    ok = (flat >= 0) & (flat < E)
    order = torch.sort(torch.where(ok, flat, torch.full_like(flat, E)), stable=True)[1]
    n = int(ok.sum())
    assert torch.equal(p.order.cpu().long()[:n], order[:n])
    assert bool((p.order[n:] == -1).all())
    position = torch.full_like(flat, -1)
    position[order[:n]] = torch.arange(n)
    assert torch.equal(p.position.cpu().long().reshape(-1), position)
    counts = torch.bincount(flat[ok], minlength=E)
    assert p.offsets.cpu().tolist() == [0] + torch.cumsum(counts, 0).tolist()


# ---------------------------------------------------------------- the join

@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,k,N", [(1, 1, 1), (5, 3, 7), (33, 2, 256), (700, 4, 100), (9, 8, 1023), (64, 32, 8)])
def test_combine_and_its_gradient(dev, T, k, N, dt):
    from nerfhip import experts
    g = torch.Generator().manual_seed(N)
    E = 6
    e = torch.randint(0, E, (T, k), generator=g, dtype=torch.int32)
    e[torch.rand(T, k, generator=g) < 0.2] = -1
    p = experts.plan(e.to(dev), E)
    y = torch.randn(T * k, N, generator=g).to(dt)
    w = torch.randn(T, k, generator=g)
    dout = torch.randn(T, N, generator=g).to(dt)
    yl, wl = y.to(dev).requires_grad_(), w.to(dev).requires_grad_()
    out = experts.combine(yl, wl, p)
    dy, dw = torch.autograd.grad(out, [yl, wl], dout.to(dev))
    pos = p.position.cpu().long()
    rows = torch.where((pos >= 0)[..., None], y.double()[pos.clamp_min(0)], torch.zeros((), dtype=torch.float64))
    terms = w.double()[..., None] * rows
    want, size = terms.sum(1), terms.abs().sum(1)
    assert bool(((out.detach().cpu().double() - want).abs() <= (k + 1) * 2.0 ** -23 * size + HALF_STEP[dt] * want.abs() + 1e-7).all())
    wdw = (rows * dout.double()[:, None]).sum(-1)
    sdw = (rows * dout.double()[:, None]).abs().sum(-1)
    assert bool(((dw.cpu().double() - wdw).abs() <= (N + 8) * 2.0 ** -23 * sdw).all())
    wdy = torch.zeros(T * k, N, dtype=torch.float64)
    live = pos >= 0
    wdy[pos[live]] = (w.double()[..., None] * dout.double()[:, None])[live]
    assert bool(((dy.cpu().double() - wdy).abs() <= (2.0 ** -24 + HALF_STEP[dt]) * wdy.abs() + 2.0 ** -25).all())
    # each gradient alone
    (only_y,) = torch.autograd.grad(experts.combine(yl, w.to(dev), p), yl, dout.to(dev))
    (only_w,) = torch.autograd.grad(experts.combine(y.to(dev), wl, p), wl, dout.to(dev))
    assert torch.equal(only_y, dy) and torch.equal(only_w, dw)


def test_a_trained_gate_end_to_end(dev):
    """Gate, plan, torch experts on the sorted rows, join: gradients of gate and experts against
    64-bit autograd of the dense form."""
    from nerfhip import experts
    g = torch.Generator().manual_seed(5)
    T, E, k, D = 96, 6, 2, 16
    x, gate = torch.randn(T, D, generator=g), torch.randn(E, D, generator=g)
    ws = torch.randn(E, D, D, generator=g) * D ** -0.5
    gl, wl = gate.to(dev).requires_grad_(), ws.to(dev).requires_grad_()
    xd = x.to(dev)
    w, e = experts.route(xd @ gl.t(), k)
    p = experts.plan(e, E)
    rows = xd[(p.order // k).long()]
    held = e.reshape(-1)[p.order.long()].long()
    y = torch.relu((wl[held] @ rows[:, :, None])[..., 0])
    out = experts.combine(y, w, p)
    dg, dws = torch.autograd.grad((out ** 2).sum(), [gl, wl])
    g64, w64 = gate.double().requires_grad_(), ws.double().requires_grad_()
    s = torch.softmax(x.double() @ g64.t(), 1)
    c = torch.gather(s, 1, e.cpu().long())
    c = c / c.sum(1, keepdim=True)
    ys = torch.relu(torch.matmul(w64[e.cpu().long()], x.double()[:, None, :, None])[..., 0])
    ref = (c[..., None] * ys).sum(1)
    rg, rw = torch.autograd.grad((ref ** 2).sum(), [g64, w64])
    for got, want in ((dg, rg), (dws, rw)):
        assert float((got.cpu().double() - want).norm() / want.norm()) < 1e-5


def test_a_captured_training_step_replays(dev):
    """Gate, plan, join and their backward in one graph (torch.autograd.grad), with eager work and
    synchronisation between the replays, against eager steps."""
    from nerfhip import experts
    T, E, k, N = 300, 10, 3, 48
    logits = [torch.randn(T, E, device=dev) for _ in range(3)]
    ys = [torch.randn(T * k, N, device=dev).bfloat16() for _ in range(3)]
    douts = [torch.randn(T, N, device=dev).bfloat16() for _ in range(3)]

    def step(l, y, d):
        w, e = experts.route(l, k, score="sigmoid", groups=5, top_groups=2)
        p = experts.plan(e, E)
        out = experts.combine(y, w, p)
        return (e, out.detach(), *torch.autograd.grad(out, [l, y], d))

    want = [step(l.clone().requires_grad_(), y.clone().requires_grad_(), d) for l, y, d in zip(logits, ys, douts)]
    l, y, d = logits[0].clone().requires_grad_(), ys[0].clone().requires_grad_(), douts[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(l, y, d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(l, y, d)
    for _ in range(2):
        for i in range(3):
            with torch.no_grad():
                l.copy_(logits[i])
                y.copy_(ys[i])
            d.copy_(douts[i])
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want[i]))
            step(logits[2].clone().requires_grad_(), ys[2].clone().requires_grad_(), douts[2])


def test_large_numbers_of_rows_and_a_long_row(dev):
    """Every row of a long batch, spread over many workgroups, and slots past 2^16 of one expert."""
    from nerfhip import experts
    T, E = 200003, 6
    x = torch.randn(T, E, generator=torch.Generator().manual_seed(8)).half()
    bias = torch.tensor([0.0, 0.5, -0.25, 0.125, 0.0, 0.3])
    w, e = experts.route(x.to(dev), 2, score="sigmoid", bias=bias.to(dev))
    want = ref_choice(x, 2, "sigmoid", bias, 1, 1, "max")
    assert torch.equal(e.cpu().long(), want)
    p = experts.plan(torch.zeros(T, 2, dtype=torch.int32, device=dev), E)
    assert p.order.tolist() == list(range(2 * T)) and p.offsets.tolist() == [0] + [2 * T] * E
