"""Gated experts and 8-bit products: what their entry points refuse (argument checks come before any GPU call,
so these run without one) and the 8-bit weight format on the CPU."""
import ctypes

import pytest
import torch

from nerfhip import _lib, experts, fp8


def weight(*shape, k=None):
    k = k or shape[-1]
    kp = -(-k // 128) * 128
    q = torch.zeros(*shape[:-1], kp, dtype=torch.uint8).view(torch.float8_e4m3fn)
    return fp8.Fp8Weight(q, torch.full((*shape[:-2], -(-shape[-2] // 128), kp // 128), 127, dtype=torch.uint8), k)


@pytest.mark.parametrize("kw", [
    dict(k=0), dict(k=9), dict(k=2, groups=3), dict(k=2, groups=0), dict(k=2, groups=2, top_groups=3),
    dict(k=5, groups=2, top_groups=1), dict(k=2, score="relu"), dict(k=2, group_score="sum"), dict(k=2, scale=0.0),
    dict(k=2, scale=float("nan")), dict(k=2, scale=float("inf")), dict(k=2, bias=torch.zeros(7)),
    dict(k=2, bias=torch.zeros(8, dtype=torch.float16))])
def test_route_refuses(kw):
    with pytest.raises(ValueError, match="route"):
        experts.route(torch.zeros(4, 8), **kw)


def test_route_refuses_shapes_and_types():
    for x in (torch.zeros(8), torch.zeros(2, 2, 8), torch.zeros(4, 8, dtype=torch.float64), torch.zeros(4, 8).int(),
              torch.zeros(4, 0), torch.zeros(4, 1025)):
        with pytest.raises(ValueError, match="route"):
            experts.route(x, 1)
    with pytest.raises(ValueError, match="route"):
        experts.route(torch.zeros(4, 64), 33)
    with pytest.raises(ValueError, match="route"):
        experts.route(torch.zeros(4, 130), 2, groups=65)


def test_no_cpu_fallback():
    e = torch.zeros(2, 1, dtype=torch.int32)
    p = experts.Plan(torch.zeros(2, dtype=torch.int32), e, torch.zeros(3, dtype=torch.int32))
    for f in (lambda: experts.route(torch.zeros(2, 2), 1), lambda: experts.plan(e, 2),
              lambda: experts.combine(torch.zeros(2, 4), torch.zeros(2, 1), p),
              lambda: experts.expert_linear(torch.zeros(2, 128), weight(2, 4, 128), p),
              lambda: fp8.linear(torch.zeros(2, 128), weight(4, 128)), lambda: fp8.quantize_weight(torch.zeros(4, 4))):
        with pytest.raises(_lib.NerfHipError, match="no CPU fallback|need tensors on a ROCm GPU"):
            f()


def test_plan_refuses():
    for e, n in ((torch.zeros(4, dtype=torch.int32), 2), (torch.zeros(4, 2), 2), (torch.zeros(4, 2).long(), 2),
                 (torch.zeros(4, 0, dtype=torch.int32), 2), (torch.zeros(4, 2, dtype=torch.int32), 0),
                 (torch.zeros(4, 2, dtype=torch.int32), 1025)):
        with pytest.raises(ValueError, match="plan"):
            experts.plan(e, n)


def test_products_and_joins_refuse():
    i = torch.int32
    p = experts.Plan(torch.zeros(6, dtype=i), torch.zeros(3, 2, dtype=i), torch.zeros(3, dtype=i))
    w = weight(2, 8, 100)
    x = torch.zeros(3, 100)
    bad = [
        lambda: experts.expert_linear(x, weight(8, 100), p, gather=True),            # one matrix
        lambda: experts.expert_linear(x, weight(3, 8, 100), p, gather=True),         # another number of experts
        lambda: experts.expert_linear(x, w, p),                                      # unsorted rows without gather
        lambda: experts.expert_linear(torch.zeros(3, 99), w, p, gather=True),
        lambda: experts.expert_linear(x.double(), w, p, gather=True),
        lambda: experts.expert_linear(x, w, p, gather=True, bias=torch.zeros(8)),
        lambda: experts.expert_linear(x, w, p._replace(order=p.order.long()), gather=True),
        lambda: experts.expert_linear(x, w, p._replace(order=p.order[:5]), gather=True),
        lambda: experts.expert_linear(x, w, p, gather=True, out_dtype=torch.float64),
        lambda: experts.expert_linear(x, w, tuple(p), gather=True),
        lambda: experts.combine(torch.zeros(5, 8), torch.zeros(3, 2), p),
        lambda: experts.combine(torch.zeros(6, 8), torch.zeros(3, 2).half(), p),
        lambda: experts.combine(torch.zeros(6, 8), torch.zeros(2, 3), p),
        lambda: experts.combine(torch.zeros(6), torch.zeros(3, 2), p),
        lambda: experts.combine(torch.zeros(6, 8).int(), torch.zeros(3, 2), p),
        lambda: fp8.linear(x, w),
        lambda: fp8.linear(x, weight(8, 100), bias=torch.zeros(8).half()),
        lambda: fp8.linear(torch.zeros(()), weight(8, 100)),
        lambda: fp8.linear(torch.zeros(3, 0), weight(8, 100)),
        lambda: fp8.linear(torch.zeros(3, 128), weight(8, 100)),
        lambda: fp8.quantize_weight(torch.zeros(4)),
        lambda: fp8.quantize_weight(torch.zeros(0, 4)),
        lambda: fp8.quantize_weight(torch.zeros(4, 4).double()),
    ]
    for k, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {k} was taken")
    with pytest.raises(_lib.NerfHipError, match="no gradient"):
        fp8.linear(torch.zeros(3, 100, requires_grad=True), weight(8, 100))


def test_weight_format():
    q = torch.zeros(130, 256, dtype=torch.float8_e4m3fn)
    s = torch.full((2, 2), 127, dtype=torch.uint8)
    assert fp8.Fp8Weight(q, s, 200).shape == (130, 200)
    assert fp8.Fp8Weight(q, s.view(torch.float8_e8m0fnu), 256).shape == (130, 256)
    for a in ((q.float(), s, 200), (q[0], s, 200), (q, s, 128), (q, s, 257), (q, s[:1], 200), (q, s.int(), 200),
              (q, s, 0), (q[:, ::2], s[:, :1].contiguous(), 128), (q[:0], s[:0], 200)):
        with pytest.raises(ValueError, match="Fp8Weight"):
            fp8.Fp8Weight(*a)
    w = fp8.Fp8Weight(torch.full((2, 128), 1.5).to(torch.float8_e4m3fn), torch.tensor([[130]], dtype=torch.uint8), 100)
    assert torch.equal(w.dequantize(), torch.full((2, 100), 12.0))
    w.scale[0, 0] = 255
    assert bool(torch.isnan(w.dequantize()).all())


def test_library_refuses_bad_descriptors():
    """(In a thread of its own: the last error is kept for each thread.)"""
    from concurrent.futures import ThreadPoolExecutor
    with ThreadPoolExecutor(1) as ex:
        ex.submit(_bad_descriptors).result()


def _bad_descriptors():
    L = _lib.lib()
    one = ctypes.c_void_p(16)       # (never read: the sizes are refused first)

    def said(rc, what):
        assert rc == 1001 and what in L.nerf_last_error().decode(), L.nerf_last_error()

    d = experts._Route(one, 8, 4, 0, 8, 9, 0, 1, 1, 0, 1, None, 1.0, one, one)
    said(L.nerf_route(ctypes.addressof(d), None), "k must be")
    d.k, d.groups = 2, 3
    said(L.nerf_route(ctypes.addressof(d), None), "groups")
    d.groups, d.type = 1, 3
    said(L.nerf_route(ctypes.addressof(d), None), "type")
    said(L.nerf_expert_plan(one, 8, 1025, one, one, one, None, 0, None), "bad size")
    said(L.nerf_expert_plan(one, 9000, 8, one, one, one, None, 0, None), "workspace")
    f = fp8._Fp8Linear(one, 128, 64, None, 0, 0, 1, 1, 0, 64, 64, 128, one, one, None, None, one, 64)
    said(L.nerf_fp8_linear(ctypes.addressof(f), None, 0, None), "workspace")
    f.E = 2
    said(L.nerf_fp8_linear(ctypes.addressof(f), None, 0, None), "offsets")
    f.E, f.x_rows = 1, 63
    said(L.nerf_fp8_linear(ctypes.addressof(f), None, 0, None), "rows of x")
    f.x_rows, f.ldo = 64, 63
    said(L.nerf_fp8_linear(ctypes.addressof(f), None, 0, None), "pitch")
    f.ldo, f.wq = 64, 8
    said(L.nerf_fp8_linear(ctypes.addressof(f), None, 0, None), "alignment")
