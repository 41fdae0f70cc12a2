"""Muon's refusals (argument checks come before any GPU call, so these run without one)."""
import ctypes

import pytest
import torch

from nerfhip import _lib, muon


def test_orthogonalize_refuses():
    for g, kw in ((torch.zeros(4), {}), (torch.zeros(4, 4).double(), {}), (torch.zeros(4, 4).int(), {}),
                  (torch.zeros(4, 4), dict(steps=0)), (torch.zeros(4, 4), dict(steps=1.5)),
                  (torch.zeros(4, 4), dict(steps=101)), (torch.zeros(4, 4), dict(eps=0.0)),
                  (torch.zeros(4, 4), dict(eps=float("nan"))), (torch.zeros(1, (1 << 20) + 1), {})):
        with pytest.raises(ValueError):
            muon.orthogonalize(g, **kw)
    with pytest.raises(_lib.NerfHipError, match="no CPU"):
        muon.orthogonalize(torch.zeros(4, 4))


def test_muon_update_refuses():
    p, q = torch.zeros(4, 6), torch.zeros(6, 4)
    bad = [(([p], [p.clone()], []), {}), (([p], [q], [p.clone()]), {}), (([p], [p.clone()], [q]), {}),
           (([p.double()], [p.clone()], [p.clone()]), {}), (([p], [p.half()], [p.clone()]), {}),
           (([q.t()], [p.clone()], [p.clone()]), {}), (([p[0]], [p[0].clone()], [p[0].clone()]), {}),
           (([p, p], [p.clone()] * 2, [p.clone(), p.clone()]), {}), (([p], [p.clone()], [p]), {}),
           (([p], [p.clone()], [p.clone()]), dict(momentum=1.0)), (([p], [p.clone()], [p.clone()]), dict(momentum=-0.1)),
           (([p], [p.clone()], [p.clone()]), dict(weight_decay=-1.0)), (([p], [p.clone()], [p.clone()]), dict(clip=-1.0)),
           (([p], [p.clone()], [p.clone()]), dict(clip=float("nan"))), (([p], [p.clone()], [p.clone()]), dict(steps=0)),
           (([p], [p.clone()], [p.clone()]), dict(lr=torch.zeros(2))),
           (([p], [p.clone()], [p.clone()]), dict(lr=torch.zeros((), dtype=torch.float64)))]
    for a, kw in bad:
        with pytest.raises(ValueError, match="muon"):
            muon.muon_update(*a, **{"lr": 0.1, **kw})
    with pytest.raises(_lib.NerfHipError, match="no CPU"):
        muon.muon_update([p], [p.clone()], [p.clone()], 0.1)
    muon.muon_update([], [], [], 0.1)
    muon.muon_update([torch.zeros(0, 4)], [torch.zeros(0, 4)], [torch.zeros(0, 4)], 0.1)


def test_hip_muon_refuses():
    w, b = torch.zeros(16, 16, requires_grad=True), torch.zeros(16, requires_grad=True)
    assert muon.is_hidden_matrix(w) and not muon.is_hidden_matrix(b) and not muon.is_hidden_matrix(torch.zeros(3, 128))
    for params, kw in (([b], {}), ([{"params": [w]}], {}), ([w], dict(muon_ratio=0.0)), ([w], dict(clip=-1.0)),
                       ([w], dict(clip=float("nan")))):
        with pytest.raises(ValueError, match="HipMuon"):
            muon.HipMuon(params, **kw)
    with pytest.raises(_lib.NerfHipError, match="no CPU"):
        muon.HipMuon([w, b])


def test_library_refuses_bad_descriptors():
    """(In a thread of its own: the last error is kept for each thread.)"""
    from concurrent.futures import ThreadPoolExecutor

    def run():
        L = _lib.lib()
        one = 16        # (never read: the sizes are refused first)
        g = (muon._Group * 1)(muon._Group(one, one, None, 4, 4, 1, 0, 0))
        o = muon._Options(0, 0, 0, 5, 0.0, 0.0, 0.0, 1e-7, -1.0, None)
        at, opt = ctypes.addressof(g), ctypes.addressof(o)

        def said(what):
            assert L.nerf_muon(at, 1, opt, None, 0, None) == 1001
            assert what in L.nerf_last_error().decode(), L.nerf_last_error()

        said("workspace")
        o.steps = 0
        said("steps")
        o.steps, o.type, o.update = 5, 1, 1
        said("type")
        o.type = 0
        said("null pointer")            # an update without a momentum
        o.update, g[0].m = 0, 0
        said("bad size")
        assert L.nerf_muon_workspace(None, 1) == 0

    with ThreadPoolExecutor(1) as ex:
        ex.submit(run).result()
