"""Muon (nerfhip/muon.py on csrc/muon_ops.hip) against 64-bit Newton-Schulz on the CPU.

Bound: one step maps singular values by p(s) = a s + b s^3 + c s^5, whose slope on [0, 1.2024] is at most
L = 4 (3.4445 at 0, 3.97 at the end), so what a step adds to the error is multiplied by at most 4 in each later one.
A step's own error is taken as e |X_k| (Frobenius) with e = 2^-19: operands of 22 bits (2^-22 each, three products
in a row with coefficients a, b, c: 10 * 2^-22 at most together), the FP32 sums below that. |X_k| <= min(L^k,
1.2024 sqrt r)."""
import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


def ref(g, steps=5, eps=1e-7):
    x = g.double()
    x = x / (x.norm() + eps)
    if g.shape[0] > g.shape[1]:
        return ref(g.t(), steps, eps).t()
    for _ in range(steps):
        a = x @ x.t()
        x = A * x + (B * a + C * (a @ a)) @ x
    return x


def bound(shape, steps=5):
    r = min(shape)
    return 2.0 ** -19 * sum(4.0 ** (steps - k) * min(4.0 ** k, 1.2024 * math.sqrt(r)) for k in range(steps + 1))


def check(got, want, steps=5):
    err = got.cpu().double() - want
    tol = bound(want.shape, steps) + HALF_STEP[got.dtype] * float(want.norm())
    if got.dtype == torch.float16:
        tol += 2.0 ** -25 * math.sqrt(want.numel())
    assert float(err.norm()) <= tol, (float(err.norm()), tol)


SHAPES = [(1, 1), (1, 7), (9, 1), (3, 5), (16, 16), (31, 33), (64, 64), (65, 63), (128, 283), (256, 63), (256, 256),
          (256, 319), (100, 1000), (700, 130), (513, 257)]


@pytest.mark.parametrize("m,n", SHAPES)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_orthogonalize(dev, m, n, dt):
    from nerfhip import muon
    g = torch.randn(m, n, generator=torch.Generator().manual_seed(m * n)).to(dt)
    check(muon.orthogonalize(g.to(dev)), ref(g))
    if m > 3:    # not contiguous
        assert torch.equal(muon.orthogonalize(g.t().contiguous().to(dev).t()), muon.orthogonalize(g.to(dev)))


def test_large_tiles(dev):
    """Enough 128 x 128 tiles for the large ones, with ragged sides."""
    from nerfhip import muon
    g = torch.randn(3, 1030, 1500, generator=torch.Generator().manual_seed(1))
    for v in (g, g.transpose(1, 2).contiguous()):
        out = muon.orthogonalize(v.to(dev))
        for i in range(3):
            check(out[i], ref(v[i]))
        # (fewer matrices may take other tiles, which add a mirrored element's terms in another order)
        check(muon.orthogonalize(v[1:2].to(dev))[0], ref(v[1]))
        assert torch.equal(out, muon.orthogonalize(v.to(dev)))


@pytest.mark.parametrize("steps", [1, 2, 7])
def test_number_of_steps_and_stacks(dev, steps):
    from nerfhip import muon
    g = torch.randn(2, 3, 40, 70, generator=torch.Generator().manual_seed(1))
    out = muon.orthogonalize(g.to(dev), steps=steps)
    for i in range(2):
        for j in range(3):
            check(out[i, j], ref(g[i, j], steps), steps)


def test_singular_values_come_near_one(dev):
    from nerfhip import muon
    g = torch.randn(96, 200, generator=torch.Generator().manual_seed(4)).to(dev)
    s = torch.linalg.svdvals(muon.orthogonalize(g).cpu().double())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.2024 + 1e-4


def test_degenerate_matrices(dev):
    from nerfhip import muon
    g = torch.randn(8, 70, 90, generator=torch.Generator().manual_seed(2))
    g[1] = 0.0
    g[2] = torch.outer(g[2, :, 0], g[2, 0])               # rank one
    g[3] = 0.0
    g[3, 5, 7] = 3.0                                      # one entry
    g[4] *= 1e25                                          # squares beyond float32
    g[5] *= 1e-3
    g[6, 3, 3] = math.nan
    g[7, 3, 3] = math.inf
    out = muon.orthogonalize(g.to(dev)).cpu()
    for i in (0, 2, 3, 4, 5):
        check(out[i], ref(g[i]))
    assert torch.equal(out[1], torch.zeros_like(out[1]))
    assert bool(torch.isnan(out[6]).all()) and bool(torch.isnan(out[7]).all())
    check(muon.orthogonalize(g[0].to(dev) * 1e-6, eps=1e-2).cpu(), ref(g[0] * 1e-6, eps=1e-2))
    assert muon.orthogonalize(torch.empty(0, 4, 5, device=dev)).shape == (0, 4, 5)


def ref_update(p, g, b, lr, mu, nesterov, wd, clip):
    g = g.double() if clip is None else g.double().clamp(-clip, clip)
    b = mu * b.double() + g
    u = g + mu * b if nesterov else b
    o = ref(u)
    return p.double() * (1 - lr * wd) - lr * math.sqrt(max(1.0, p.shape[0] / p.shape[1])) * o, b


@pytest.mark.parametrize("nesterov,wd,clip", [(True, 0.0, None), (True, 0.1, 0.5), (False, 0.01, None)])
def test_muon_update(dev, nesterov, wd, clip):
    """20 matrices (two sets of launches) of many shapes, two steps."""
    from nerfhip import muon
    gen = torch.Generator().manual_seed(7)
    shapes = SHAPES + [(40, 20), (20, 40), (33, 33), (5, 300), (300, 5)]
    ps, bs = [[torch.randn(*s, generator=gen) for s in shapes] for _ in range(2)]
    dp, db = [[t.to(dev) for t in v] for v in (ps, bs)]
    for step in range(2):
        gs = [torch.randn(*s, generator=gen) for s in shapes]
        dg = [t.to(dev) for t in gs]
        lr = 0.02 if step else torch.tensor(0.02, device=dev)
        muon.muon_update(dp, dg, db, lr, momentum=0.9, nesterov=nesterov, weight_decay=wd, clip=clip)
        for i, s in enumerate(shapes):
            want, buf = ref_update(ps[i], gs[i], bs[i], 0.02, 0.9, nesterov, wd, clip)
            assert float((db[i].cpu().double() - buf).abs().max()) <= 3 * 2.0 ** -24 * float(buf.abs().max() + 1)
            err = float((dp[i].cpu().double() - want).norm())
            assert err <= 0.02 * max(1.0, s[0] / s[1]) ** 0.5 * 2 * bound(s) + 4 * 2.0 ** -24 * float(want.norm()), s
            assert torch.equal(dg[i].cpu(), gs[i])
            ps[i], bs[i] = dp[i].cpu(), db[i].cpu()


def test_update_in_a_graph_and_on_another_stream(dev):
    """Replays with new gradients and a new learning rate equal eager steps bit for bit."""
    from nerfhip import muon
    shapes = [(256, 63), (256, 256), (128, 283)]
    p0 = [torch.randn(*s, device=dev) for s in shapes]
    gs = [[torch.randn(*s, device=dev) for s in shapes] for _ in range(4)]
    lrs = [0.02, 0.01, 0.03, 0.005]
    lr = torch.tensor(0.0, device=dev)

    def fresh():
        return [p.clone() for p in p0], [torch.zeros_like(p) for p in p0]

    pe, be = fresh()
    want = []
    for g, v in zip(gs, lrs):
        lr.fill_(v)
        muon.muon_update(pe, g, be, lr)
        want.append([p.clone() for p in pe])
    side = torch.cuda.Stream()
    ps, bs = fresh()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for g, v in zip(gs, lrs):
            lr.fill_(v)
            muon.muon_update(ps, g, bs, lr)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(ps, pe))
    pg, bg = fresh()
    g = [torch.zeros_like(p) for p in p0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon.muon_update(pg, g, bg, lr)
    for a, b in zip(pg + bg, fresh()[0] + fresh()[1]):
        a.copy_(b)
    for k in range(4):
        lr.fill_(lrs[k])
        torch._foreach_copy_(g, gs[k])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(pg, want[k])), k
        muon.orthogonalize(gs[k][0])


def _params(dev, seed=3):
    g = torch.Generator(device=dev).manual_seed(seed)
    shapes = [(256, 63), (256,), (256, 256), (1, 256), (1,), (3, 128), (128, 283), (128,), (16, 16), (15, 40)]
    return [torch.randn(s, device=dev, generator=g).requires_grad_() for s in shapes], g


def test_hip_muon_splits_the_parameters(dev):
    """Matrices as muon_update, the rest bit for bit as HipAdam alone; lr through the device tensor; a state
    dict round trip goes on as if nothing had been."""
    from nerfhip.adam import HipAdam
    from nerfhip.muon import HipMuon, is_hidden_matrix, muon_update
    pa, g = _params(dev)
    pb, _ = _params(dev)
    pc, _ = _params(dev)
    opt = HipMuon(pa, lr=1e-3, clip=20.0)
    assert [len(v["params"]) for v in opt.param_groups] == [4, 6]
    mats, rest = [p for p in pb if is_hidden_matrix(p)], [p for p in pb if not is_hidden_matrix(p)]
    adam, bufs = HipAdam(rest, lr=1e-3, clip=20.0), [torch.zeros_like(p) for p in mats]
    for step in range(6):
        if step == 3:
            again = HipMuon(pc, lr=5.0, clip=20.0)
            with torch.no_grad():
                torch._foreach_copy_(pc, pa)
            again.load_state_dict(copy.deepcopy(opt.state_dict()))   # (torch's own would share the tensors)
            for v in opt.param_groups:
                v["lr"].fill_(4e-4)
            for v in again.param_groups:
                v["lr"].fill_(4e-4)
            adam.param_groups[0]["lr"].fill_(4e-4)
        lr = torch.tensor(1e-3 if step < 3 else 4e-4, device=dev)
        for a, b, c in zip(pa, pb, pc):
            gr = torch.randn(a.shape, device=dev, generator=g) * 15.0
            a.grad, b.grad, c.grad = gr.clone(), gr.clone(), gr.clone()
        opt.step()
        adam.step()
        muon_update([p.detach() for p in mats], [p.grad for p in mats], bufs, lr * 40.0, clip=20.0)
        if step >= 3:
            again.step()
            assert all(torch.equal(a, c) for a, c in zip(pa, pc)), step
        assert all(torch.equal(a, b) for a, b in zip(pa, pb)), step
    pa[0].grad = None
    with pytest.raises(ValueError, match="no gradient"):
        opt.step()


def test_hip_muon_of_matrices_alone(dev):
    """No other parameters; a learning rate on the host, then a float; a group that was added is refused."""
    from nerfhip.muon import HipMuon
    p0, g = torch.randn(40, 30, device=dev), torch.randn(40, 30, device=dev)
    outs = []
    for lr in (None, torch.tensor(2e-3), torch.tensor(2e-3, dtype=torch.float64), 2e-3):
        p = p0.clone().requires_grad_()
        opt = HipMuon([p], lr=2e-3, weight_decay=0.1)
        if lr is not None:
            opt.param_groups[0]["lr"] = lr
        for _ in range(2):
            p.grad = g.clone()
            opt.step()
        outs.append(p.detach())
    assert all(torch.equal(outs[0], v) for v in outs[1:]) and not torch.equal(outs[0], p0)
    opt.zero_grad()
    assert opt.step() is None
    opt.add_param_group({"params": [torch.zeros(16, 16, device=dev, requires_grad=True)]})
    with pytest.raises(ValueError, match="groups"):
        opt.step()


def test_two_streams_at_once(dev):
    """Steps of two optimisers' matrices and an orthogonalisation on two streams, nothing waiting between: as one
    after the other."""
    from nerfhip import muon
    ga = [torch.randn(2, 300, 500, device=dev) for _ in range(6)]
    gb = [torch.randn(5, 100, 40, device=dev) for _ in range(6)]
    want = [(muon.orthogonalize(a), muon.orthogonalize(b)) for a, b in zip(ga, gb)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for a, b in zip(ga, gb):
        with torch.cuda.stream(s1):
            x = muon.orthogonalize(a)
        with torch.cuda.stream(s2):
            y = muon.orthogonalize(b)
        got.append((x, y))
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) and torch.equal(b, d) for (a, b), (c, d) in zip(got, want))


@pytest.mark.parametrize("n_importance", [128, 0])
def test_trainer_steps_with_muon(dev, n_importance):
    """NerfTrainer(adam="muon"): graph steps (two eager, the capture, replays) equal eager ones bit for bit, the
    matrices move by 40 lr times a nearly orthogonal matrix, and lr 0 moves nothing."""
    from goldlib import load, params_of
    from nerfhip.train import NerfTrainer
    z = load("t1_train_step")
    g = torch.Generator(device=dev).manual_seed(1)
    n = 256
    ro = torch.randn(n, 3, device=dev, generator=g) * 0.1 + torch.tensor([0.0, 0.0, 4.0], device=dev)
    rd = torch.nn.functional.normalize(torch.randn(n, 3, device=dev, generator=g) * 0.2 -
                                       torch.tensor([0.0, 0.0, 1.0], device=dev), dim=-1)
    gt = torch.rand(n, 3, device=dev, generator=g)
    runs = []
    for graph in (False, True):
        torch.manual_seed(5)
        tr = NerfTrainer(dev, params_of(z), N_importance=n_importance, graph=graph, adam="muon", lr=1e-4)
        first = {k: v.clone() for k, v in tr.state().items()}
        losses = [tr.step(ro, rd, gt)["loss"].item() for _ in range(6)]
        runs.append((losses, {k: v.clone() for k, v in tr.state().items()}, tr))
    assert runs[0][0] == runs[1][0]
    for k, v in runs[0][1].items():
        assert torch.equal(v, runs[1][1][k]), k
    tr = runs[1][2]
    moved = (runs[0][1]["model.pts_linears.2.weight"] - first["model.pts_linears.2.weight"]).norm()
    assert 0 < float(moved) <= 6 * 40 * 1e-4 * 1.2024 * 16      # six steps of at most 1.2024 sqrt(256)
    tr.set_lr(0.0)
    before = [p.detach().clone() for p in tr.trained_parameters()]
    tr.step(ro, rd, gt)
    assert all(torch.equal(a, b) for a, b in zip(before, tr.trained_parameters()))
