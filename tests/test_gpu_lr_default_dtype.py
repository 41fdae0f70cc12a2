"""A learning rate that someone set as a number becomes one float32 on the device, whatever torch's default type is
(the kernels read four bytes)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[torch.bfloat16, torch.float16, torch.float64], ids=str)
def default_dtype(request):
    was = torch.get_default_dtype()
    torch.set_default_dtype(request.param)
    yield request.param
    torch.set_default_dtype(was)


@pytest.mark.parametrize("lr", [0.0009765625, torch.tensor(0.0009765625, dtype=torch.float64)], ids=["number", "tensor"])
@pytest.mark.parametrize("kind", ["adam", "muon"])
def test_a_number_as_learning_rate(default_dtype, kind, lr):
    from nerfhip.adam import HipAdam
    from nerfhip.muon import HipMuon
    dev = torch.device("cuda:0")
    shapes = [(40, 30), (30,)]
    start = [torch.randn(s, device=dev, dtype=torch.float32) for s in shapes]
    grads = [torch.randn(s, device=dev, dtype=torch.float32) for s in shapes]
    runs = []
    for given in (None, lr):
        ps = [p.clone().requires_grad_() for p in start]
        opt = (HipAdam if kind == "adam" else HipMuon)(ps, lr=0.0009765625)
        for _ in range(2):
            for p, g in zip(ps, grads):
                p.grad = g.clone()
            if given is not None:
                for v in opt.param_groups:
                    v["lr"] = given
            opt.step()
            for v in opt.param_groups:
                assert v["lr"].dtype == torch.float32 and v["lr"].device == ps[0].device
        runs.append(ps)
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    assert not any(torch.equal(a, b) for a, b in zip(runs[0], start))
