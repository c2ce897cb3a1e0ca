"""Norm, codes, a projection on them, the router's scores, routing and experts, one after another as a layer runs them."""
import numpy as np
import pytest
import torch

from tests import ffn_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mld():
    import __graft_entry__ as g
    return g.import_package()


def _matrix(packed, scales, o, i, bits):
    p = packed.cpu().numpy().reshape(-1)
    if bits == 4:
        p = np.stack((p & 15, p >> 4), -1).reshape(-1)
    w = p.reshape(i // 4, o // 4, 4, 4).transpose(1, 3, 0, 2).reshape(o, i).astype(np.float64) - (8 if bits == 4 else 128)
    s = scales.cpu().numpy().astype(np.float64)
    return w * np.repeat(s, i // s.shape[0], 0).T


@pytest.mark.parametrize("n", [1, 3, 40, 200])
@pytest.mark.parametrize("captured", [False, True])
def test_a_layer(mld, n, captured):
    from examples import expert_layer as ex
    gen = torch.Generator(device="cuda").manual_seed(n)
    d, f, e, k, o = 256, 128, 16, 3, 320
    layer = ex.ExpertLayer(mld, gen, d, f, e, k, o, max_tokens=max(n, 20))
    start = torch.randn(n, d, generator=gen, device="cuda").half()
    attention = torch.randn(n, d, generator=gen, device="cuda").half()
    stream = start.clone()
    if captured:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            layer.run(attention, stream)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                out = layer.run(attention, stream)
            for _ in range(3):
                stream.copy_(start)
                graph.replay()
        s.synchronize()
    else:
        out = layer.run(attention, stream)
    torch.cuda.synchronize()
    assert layer.experts.device_status() == 0 and layer.project.device_status() == 0
    h, v, rstd = ref.add_norm(attention.cpu().numpy(), start.cpu().numpy(), layer.norm.cpu().numpy(), 1e-6, 0.0)
    q, step, _ = ref.codes(v, rstd, True)
    assert np.array_equal(layer.codes[:n].cpu().numpy(), q)
    w = _matrix(layer.project_w[0], layer.project_w[1], o, d, 8)
    want = (q * step) @ w.T
    size = np.abs(q * step) @ np.abs(w).T
    assert (np.abs(out.cpu().numpy() - want) <= 2.0 ** -11 * np.abs(want) + 80 * 2.0 ** -24 * size + 2.0 ** -24).all()
    # what follows is taken from what the steps before gave, so that each is held to its own errors
    y, logits = layer.y[:n].cpu().numpy(), layer.logits[:n].cpu().numpy()
    ids, gates = ref.route(logits, layer.balance.cpu().numpy(), k, True, 1, 1, 1, True, 1.5)
    assert np.array_equal(layer.ids[:n].cpu().numpy(), ids)
    assert np.allclose(layer.gates[:n].cpu().numpy(), gates, rtol=1e-5, atol=0)
    first = np.stack([_matrix(layer.weights[0][j], layer.weights[1][j], 2 * f, d, 4) for j in range(e)])
    second = np.stack([_matrix(layer.weights[2][j], layer.weights[3][j], d, f, 4) for j in range(e)])
    want, size = ref.experts(y, ids, layer.gates[:n].cpu().numpy(), first, second, h, False)
    got = stream.cpu().numpy().astype(np.float64)
    bound = ref.experts_bound(want, size, n * k > 8 * e)
    assert (np.abs(got - want) <= bound).all(), np.max(np.abs(got - want) / bound)


def test_the_example_runs(mld):
    from examples import expert_layer as ex
    layers, stream = ex.main(["--tokens", "17", "--layers", "2"])
    assert torch.isfinite(stream).all() and len(layers) == 2
