"""Every form of the 8-bit product and of Muon's products in a captured graph: replays with other inputs, eager work
and synchronisation between them, equal eager calls bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


def replays(call, inputs, other):
    want = [[t.clone() for t in call(*v)] for v in inputs]
    static = [t.clone() for t in inputs[0]]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = call(*static)
    for _ in range(2):
        for v, w in zip(inputs, want):
            for s, t in zip(static, v):
                s.copy_(t)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, w))
            other()


@pytest.mark.parametrize("M,N,K,out", [(1, 200, 300, torch.bfloat16), (30, 200, 300, torch.float32), (500, 300, 700, torch.float32),
                                       (3000, 1500, 700, torch.bfloat16), (33000, 200, 250, torch.bfloat16),
                                       (33000, 200, 100, torch.float32), (5900, 5700, 4200, torch.float16)])
def test_linear(dev, M, N, K, out):
    from nerfhip import fp8
    ws = [torch.randn(N, K, device=dev) for _ in range(2)]
    xs = [torch.randn(M, K, device=dev).bfloat16() for _ in range(2)]
    f = fp8.quantize_weight(ws[0])

    def call(x, w):         # the weights are rounded in the graph, too
        return (fp8.linear(x, fp8.quantize_weight(w), relu=True, out_dtype=out),)

    replays(call, list(zip(xs, ws)), lambda: fp8.linear(xs[1], f))


@pytest.mark.parametrize("T,k,E", [(40, 2, 64), (3000, 3, 7)])
def test_experts(dev, T, k, E):
    from nerfhip import experts, fp8
    f = fp8.quantize_weight(torch.randn(E, 130, 260, device=dev))
    bias = 0.1 * torch.randn(E, device=dev)
    xs = [(torch.randn(T, 260, device=dev), torch.randn(T, E, device=dev)) for _ in range(3)]
    xs[2][1][:, 1:] = -float("inf")      # one expert for nearly all

    def call(x, l):
        w, e = experts.route(l, k, score="sigmoid", bias=bias)
        p = experts.plan(e, E)
        y = experts.expert_linear(x, f, p, gather=True)
        return (w, e, y, experts.combine(y, w, p), *p)

    replays(call, xs, lambda: call(*xs[1]))


@pytest.mark.parametrize("shape", [(3, 40, 70), (3, 1030, 1500)])
def test_orthogonalize(dev, shape):
    from nerfhip import muon
    gs = [torch.randn(*shape, device=dev) * s for s in (1.0, 1e-10, 1e-20)]
    gs[2][1] = 0.0
    replays(lambda g: (muon.orthogonalize(g),), [(g,) for g in gs], lambda: muon.orthogonalize(gs[1]))
