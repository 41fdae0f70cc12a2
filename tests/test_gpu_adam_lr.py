"""HipAdam's learning rate as someone else may leave it: the kernel reads one float32 on the device."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lr", [torch.tensor(1e-3), torch.tensor(1e-3, dtype=torch.float64), 1e-3])
def test_a_learning_rate_from_elsewhere_is_brought_to_the_device(lr):
    from nerfhip.adam import HipAdam
    dev = torch.device("cuda:0")
    p0, g = torch.randn(300, device=dev), torch.randn(300, device=dev)
    a, b = p0.clone().requires_grad_(), p0.clone().requires_grad_()
    oa, ob = HipAdam([a], lr=1e-3), HipAdam([b], lr=5.0)
    ob.param_groups[0]["lr"] = lr
    for _ in range(2):
        a.grad, b.grad = g.clone(), g.clone()
        oa.step()
        ob.step()
    assert torch.equal(a, b)
    assert ob.param_groups[0]["lr"].is_cuda and ob.param_groups[0]["lr"].dtype == torch.float32
