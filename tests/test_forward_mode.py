"""Forward-mode derivatives: gate, join and 8-bit products have none, so a dual number is refused and not stripped
of its tangent (checks come before any GPU call, so these run without one)."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from nerfhip import _lib, experts, fp8


def weight(*shape):
    q = torch.zeros(*shape, dtype=torch.uint8).view(torch.float8_e4m3fn)
    return fp8.Fp8Weight(q, torch.full((*shape[:-2], 1, shape[-1] // 128), 127, dtype=torch.uint8), shape[-1])


def calls():
    i = torch.int32
    p = experts.Plan(torch.zeros(2, dtype=i), torch.zeros(2, 1, dtype=i), torch.zeros(3, dtype=i))
    return {
        "route": (lambda v: experts.route(v, 1), (2, 4)),
        "combine's rows": (lambda v: experts.combine(v, torch.zeros(2, 1), p), (2, 8)),
        "combine's weights": (lambda v: experts.combine(torch.zeros(2, 8), v, p), (2, 1)),
        "expert_linear": (lambda v: experts.expert_linear(v, weight(2, 4, 128), p), (2, 128)),
        "expert_linear's bias": (lambda v: experts.expert_linear(torch.zeros(2, 128), weight(2, 4, 128), p, bias=v), (2, 4)),
        "linear": (lambda v: fp8.linear(v, weight(4, 128)), (3, 128)),
        "linear's bias": (lambda v: fp8.linear(torch.zeros(3, 128), weight(4, 128), bias=v), (4,)),
    }


@pytest.mark.parametrize("name", list(calls()))
@pytest.mark.parametrize("grad", [False, True])
def test_dual_numbers_are_refused(name, grad):
    f, shape = calls()[name]
    x = torch.randn(shape)
    with fwd.dual_level():
        d = fwd.make_dual(x.requires_grad_() if grad else x, torch.ones(shape))
        with pytest.raises(_lib.NerfHipError, match="forward-mode"), torch.set_grad_enabled(grad):
            f(d)
        # a plain number inside a dual level is taken as ever
        with pytest.raises(_lib.NerfHipError, match="no CPU|ROCm GPU"), torch.no_grad():
            f(torch.zeros(shape))
    with pytest.raises(_lib.NerfHipError, match="no CPU|ROCm GPU"), torch.no_grad():
        f(torch.zeros(shape))


def test_jvp_is_refused():
    with pytest.raises(_lib.NerfHipError, match="forward-mode"):
        torch.func.jvp(lambda v: experts.route(v, 1)[0], (torch.randn(2, 4),), (torch.ones(2, 4),))
