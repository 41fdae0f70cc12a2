"""Optimizer steps write parameters behind torch's back; whoever watches a tensor's version counter (the
Renderer's packed weights, autograd's check of saved tensors) has to see them."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


def test_steps_raise_the_versions_of_what_they_write(dev):
    from nerfhip.adam import HipAdam
    from nerfhip.muon import HipMuon, muon_update
    p, g, b = (torch.randn(20, 30, device=dev) for _ in range(3))
    was = [t._version for t in (p, g, b)]
    muon_update([p], [g], [b], 0.01, clip=0.1)
    assert p._version > was[0] and b._version > was[2] and g._version == was[1]
    for clip in (None, 0.5):
        for make in (HipMuon, HipAdam):
            ps = [torch.randn(20, 30, device=dev).requires_grad_(), torch.randn(30, device=dev).requires_grad_()]
            opt = make(ps, clip=clip)
            for _ in range(2):
                for q in ps:
                    q.grad = torch.randn_like(q)
                was = [q._version for q in ps]
                opt.step()
                assert all(q._version > w for q, w in zip(ps, was)), (make, clip)
            state = [t._version for s in opt.state.values() for t in s.values()]
            grad = ps[1].grad._version      # (HipAdam's part: clamped in place)
            opt.step()
            assert all(t._version > w for t, w in zip((t for s in opt.state.values() for t in s.values()), state))
            assert (ps[1].grad._version > grad) == (clip is not None)


@pytest.mark.parametrize("kind", ["muon_update", "HipMuon", "HipAdam"])
def test_a_backward_pass_over_stepped_weights_is_refused(dev, kind):
    from nerfhip.adam import HipAdam
    from nerfhip.muon import HipMuon, muon_update
    p = torch.randn(20, 30, device=dev).requires_grad_()
    x = torch.randn(5, 20, device=dev).requires_grad_()
    out = (x @ p).sum()
    p.grad = torch.randn_like(p)
    if kind == "muon_update":
        muon_update([p.detach()], [p.grad], [torch.zeros_like(p)], 0.01)
    else:
        (HipMuon if kind == "HipMuon" else HipAdam)([p]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()


def test_steps_on_inference_tensors(dev):
    """(They have no version counter.)"""
    from nerfhip.muon import muon_update
    with torch.inference_mode():
        p, g, b = (torch.randn(20, 30, device=dev) for _ in range(3))
        q, c = p.clone(), b.clone()
        muon_update([p], [g], [b], 0.01)
    q, c = q.clone(), c.clone()
    muon_update([q], [g], [c], 0.01)
    assert torch.equal(p, q) and torch.equal(b, c)


@pytest.mark.parametrize("kind", ["HipMuon", "HipAdam"])
def test_the_renderer_sees_a_step(dev, kind):
    """Render, step, render: the second image is the one of a Renderer that never saw the first weights."""
    from goldlib import load, params_of
    from nerfhip.adam import HipAdam
    from nerfhip.muon import HipMuon
    from nerfhip.synthetic import load_into_network
    from src.config import cfg, reset
    from src.models.nerf.network import Network
    from src.models.nerf.renderer.volume_renderer import Renderer
    z = load("f1_c2_crop")
    reset()
    try:
        cfg.task_arg.perturb = 0
        cfg.enable_ess = False
        cfg.enable_ert = False
        net = Network().to(dev)
        load_into_network(net, params_of(z))
        net.eval()
        rend = Renderer(net)
        batch = {"H": int(z["H"]), "W": int(z["W"]), "pose": torch.from_numpy(z["pose"])[None],
                 "intrinsics": torch.from_numpy(z["K"])[None]}
        ps = list(net.parameters())
        opt = (HipMuon if kind == "HipMuon" else HipAdam)(ps, lr=2e-3)
        gen = torch.Generator(device=dev).manual_seed(1)
        with torch.no_grad():
            before = rend.render(batch)["rgb_map"].cpu().numpy()
        for p in ps:
            p.grad = torch.randn(p.shape, device=dev, generator=gen)
        opt.step()
        with torch.no_grad():
            after = rend.render(batch)["rgb_map"].cpu().numpy()
            fresh = Renderer(net).render(batch)["rgb_map"].cpu().numpy()
    finally:
        reset()
    assert np.array_equal(after, fresh)
    assert not np.array_equal(after, before)


@pytest.mark.parametrize("adam", ["hip", "muon"])
def test_a_replayed_training_step_raises_the_versions(dev, adam):
    from goldlib import load, params_of
    from nerfhip.train import NerfTrainer
    z = load("t1_train_step")
    g = torch.Generator(device=dev).manual_seed(1)
    n = 256
    ro = torch.randn(n, 3, device=dev, generator=g) * 0.1 + torch.tensor([0.0, 0.0, 4.0], device=dev)
    rd = torch.nn.functional.normalize(torch.randn(n, 3, device=dev, generator=g) * 0.2 -
                                       torch.tensor([0.0, 0.0, 1.0], device=dev), dim=-1)
    gt = torch.rand(n, 3, device=dev, generator=g)
    tr = NerfTrainer(dev, params_of(z), graph=True, adam=adam)
    for step in range(5):       # two eager ones, the capture with its replay, two replays
        was = [p._version for p in tr.trained_parameters()]
        tr.step(ro, rd, gt)
        assert all(p._version > w for p, w in zip(tr.trained_parameters(), was)), step
