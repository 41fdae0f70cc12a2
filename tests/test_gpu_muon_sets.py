"""Lists of more matrices than one set of launches takes (32): the second set's workspace and workgroups."""
import pytest
import torch

from test_gpu_muon import bound, ref_update

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


@pytest.mark.parametrize("count", [32, 33, 70])
def test_many_matrices(dev, count):
    from nerfhip import muon
    gen = torch.Generator().manual_seed(count)
    shapes = [(1 + 7 * i % 90, 1 + 13 * i % 110) for i in range(count)]
    ps, gs, bs = [[torch.randn(*s, generator=gen) for s in shapes] for _ in range(3)]
    dp, dg, db = [[t.to(dev) for t in v] for v in (ps, gs, bs)]
    muon.muon_update(dp, dg, db, 0.02, momentum=0.9, weight_decay=0.1)
    for i, s in enumerate(shapes):
        want, buf = ref_update(ps[i], gs[i], bs[i], 0.02, 0.9, True, 0.1, None)
        assert float((db[i].cpu().double() - buf).abs().max()) <= 3 * 2.0 ** -24 * float(buf.abs().max() + 1)
        err = float((dp[i].cpu().double() - want).norm())
        assert err <= 0.02 * max(1.0, s[0] / s[1]) ** 0.5 * 2 * bound(s) + 4 * 2.0 ** -24 * float(want.norm()), (i, s)
    # one at a time: the same numbers where the tiles are the same (all of these are small)
    one = [t.to(dev) for t in ps]
    ob = [t.to(dev) for t in bs]
    for p, g, b in zip(one, dg, ob):
        muon.muon_update([p], [g], [b], 0.02, momentum=0.9, weight_decay=0.1)
    assert all(torch.equal(a, b) for a, b in zip(one, dp)) and all(torch.equal(a, b) for a, b in zip(ob, db))
