"""Experts' gated networks over packed weights against the formulas in 64 bits, on both paths."""
import functools

import numpy as np
import pytest
import torch

from tests import ffn_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mld():
    import __graft_entry__ as g
    return g.import_package()


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


@functools.lru_cache(4)
def _weights(e, d, f, bits, block):
    rng = np.random.default_rng(e * d + f)
    first, second = [ref.matrix(rng, 2 * f, d, bits, block) for _ in range(e)], [ref.matrix(rng, d, f, bits, block) for _ in range(e)]
    host = [np.stack([m[2] for m in ms]) for ms in (first, second)]
    dev = [_dev(np.stack([m[i] for m in ms])) for ms in (first, second) for i in range(2)]
    return host, dev


_bound = ref.experts_bound


def _run(mld, n, e, k, d, f, bits, block, gelu, path, ids, residual=True, seed=0):
    rng = np.random.default_rng(seed + n)
    (first, second), (w1, s1, w2, s2) = _weights(e, d, f, bits, block)
    x = rng.standard_normal((n, d)).astype(np.float16)
    weights = rng.random((n, k)).astype(np.float32)
    res = (2 * rng.standard_normal((n, d))).astype(np.float16) if residual else None
    plan = mld.MoeExperts(e, k, d, f, weight_bits=bits, block=block, activation=mld.MOE_GELU_TANH if gelu else mld.MOE_SILU, max_tokens=n,
                          force_path=path)
    out = torch.full((n, d), 7.0, dtype=torch.float16, device="cuda")
    xd, idd, wd, rd = _dev(x), _dev(ids.astype(np.int32)), _dev(weights), _dev(res) if residual else None
    plan.run(xd, idd, wd, w1, s1, w2, s2, out, residual=rd)
    torch.cuda.synchronize()
    assert plan.device_status() == 0
    want, size = ref.experts(x, ids, weights, first, second, res, gelu)
    got = out.cpu().numpy().astype(np.float64)
    bound = _bound(want, size, path == mld.MOE_PATH_MANY_ROWS)
    assert (np.abs(got - want) <= bound).all(), np.max(np.abs(got - want) / bound)
    again = torch.empty_like(out)
    plan.run(xd, idd, wd, w1, s1, w2, s2, again, residual=rd)
    assert torch.equal(out, again)  # the same bits
    return got


def _ids(rng, n, e, k, skew=0.0):
    ids = np.argsort(-(rng.standard_normal((n, e)) + skew * rng.standard_normal(e)), 1)[:, :k]
    return ids


SHAPES = [  # experts, top_k, d, f, bits, block
    (4, 2, 256, 128, 4, 32), (8, 3, 160, 96, 4, 32), (5, 1, 96, 352, 8, 0), (6, 2, 128, 64, 8, 64), (3, 3, 384, 256, 4, 128), (4, 2, 64, 32, 4, 0)]


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 33, 100])
@pytest.mark.parametrize("e,k,d,f,bits,block", SHAPES)
@pytest.mark.parametrize("path", ["few", "many"])
def test_experts(mld, n, e, k, d, f, bits, block, path):
    rng = np.random.default_rng(n * d + f)
    _run(mld, n, e, k, d, f, bits, block, n % 2 == 1, mld.MOE_PATH_FEW_ROWS if path == "few" else mld.MOE_PATH_MANY_ROWS,
         _ids(rng, n, e, k, 1.0), residual=n % 3 != 0)


@pytest.mark.parametrize("path", ["few", "many"])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_no_expert_the_same_expert_twice_and_all_on_one(mld, n, path):
    path = mld.MOE_PATH_FEW_ROWS if path == "few" else mld.MOE_PATH_MANY_ROWS
    e, k, d, f = 4, 3, 128, 64
    rng = np.random.default_rng(n)
    ids = _ids(rng, n, e, k)
    ids[0] = (2, 2, 2)
    _run(mld, n, e, k, d, f, 4, 32, False, path, ids)
    ids[n // 2:] = -1
    ids[-1, 0], ids[0, 1] = 4, 1 << 30
    _run(mld, n, e, k, d, f, 4, 32, False, path, ids)
    got = _run(mld, n, e, k, d, f, 4, 32, False, path, np.full((n, k), -5), residual=False)
    assert not got.any()
    _run(mld, n, e, k, d, f, 4, 32, True, path, np.full((n, k), 3))


@pytest.mark.parametrize("n", [300, 700])
def test_many_rows_ragged(mld, n):
    rng = np.random.default_rng(n)
    ids = _ids(rng, n, 4, 2, 1.5)
    ids[5::17] = -1
    _run(mld, n, 4, 2, 256, 128, 4, 32, False, mld.MOE_PATH_MANY_ROWS, ids)
    _run(mld, n, 5, 1, 96, 352, 8, 0, True, mld.MOE_PATH_MANY_ROWS, _ids(rng, n, 5, 1, 2.0))


@pytest.mark.parametrize("path", ["few", "many"])
def test_strides_in_place_capture_and_a_smaller_call(mld, path):
    path = mld.MOE_PATH_FEW_ROWS if path == "few" else mld.MOE_PATH_MANY_ROWS
    e, k, d, f, n = 4, 2, 256, 128, 50
    rng = np.random.default_rng(1)
    (first, second), (w1, s1, w2, s2) = _weights(e, d, f, 4, 32)
    wide = torch.from_numpy(rng.standard_normal((n, d + 40)).astype(np.float16)).cuda()
    x = wide[:, 8:8 + d]
    stream = torch.from_numpy(rng.standard_normal((n, d + 16)).astype(np.float16)).cuda()
    res = stream[:, 16:]
    start = stream.clone()
    ids, weights = _dev(_ids(rng, n, e, k).astype(np.int32)), _dev(rng.random((n, k)).astype(np.float32))
    plan = mld.MoeExperts(e, k, d, f, max_tokens=n, force_path=path)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        plan.run(x, ids, weights, w1, s1, w2, s2, res, residual=res)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            plan.run(x, ids, weights, w1, s1, w2, s2, res, residual=res)
        for rows in (n, 13):  # replayed, and a call of fewer tokens in between
            stream.copy_(start)
            if rows == n:
                graph.replay()
            else:
                plan.run(x[:rows], ids[:rows], weights[:rows], w1, s1, w2, s2, res[:rows], residual=res[:rows])
            s.synchronize()
            want, size = ref.experts(x.cpu().numpy()[:rows], ids.cpu().numpy()[:rows], weights.cpu().numpy()[:rows], first, second,
                                     start.cpu().numpy()[:rows, 16:], False)
            got = res.cpu().numpy().astype(np.float64)
            assert (np.abs(got[:rows] - want) <= _bound(want, size, path == mld.MOE_PATH_MANY_ROWS)).all()
            assert torch.equal(stream[:, :16], start[:, :16]) and torch.equal(stream[rows:], start[rows:])
        stream.copy_(start)
        graph.replay()
        s.synchronize()
    assert plan.device_status() == 0


def test_values_that_are_not_numbers_stay_with_their_token(mld):
    e, k, d, f, n = 4, 2, 128, 64, 20
    rng = np.random.default_rng(2)
    (_, _), (w1, s1, w2, s2) = _weights(e, d, f, 4, 32)
    x = rng.standard_normal((n, d)).astype(np.float16)
    ids = _ids(rng, n, e, k).astype(np.int32)
    weights = rng.random((n, k)).astype(np.float32)
    for path in (mld.MOE_PATH_FEW_ROWS, mld.MOE_PATH_MANY_ROWS):
        plan = mld.MoeExperts(e, k, d, f, max_tokens=n, force_path=path)
        outs = []
        for bad in (False, True):
            y = x.copy()
            if bad:
                y[7, 5], y[11] = np.nan, np.inf
            out = torch.empty(n, d, dtype=torch.float16, device="cuda")
            plan.run(_dev(y), _dev(ids), _dev(weights), w1, s1, w2, s2, out)
            outs.append(out.cpu().numpy())
        assert np.isnan(outs[1][7]).all() and np.isnan(outs[1][11]).all()
        rest = [t for t in range(n) if t not in (7, 11)]
        assert np.array_equal(outs[0][rest], outs[1][rest])


@pytest.mark.parametrize("path", ["few", "many"])
@pytest.mark.parametrize("n,e,k,d,f,bits,block", [(3, 1, 1, 16384, 32, 4, 32), (2, 2, 1, 32, 16384, 8, 0), (5, 1024, 32, 32, 32, 4, 32),
                                                  (2500, 7, 4, 64, 32, 4, 0), (70, 300, 1, 32, 64, 8, 32)])
def test_the_ends_of_the_ranges(mld, n, e, k, d, f, bits, block, path):
    """Long rows, many inputs, many experts, more pairs than one block orders."""
    rng = np.random.default_rng(n + e)
    ids = _ids(rng, n, e, k, 1.0)
    ids[n // 2::9] = -1
    _run(mld, n, e, k, d, f, bits, block, False, mld.MOE_PATH_FEW_ROWS if path == "few" else mld.MOE_PATH_MANY_ROWS, ids)


def test_the_path_changes_with_the_tokens_of_a_call(mld):
    e, k, d, f, n = 4, 2, 128, 64, 60
    rng = np.random.default_rng(4)
    (first, second), (w1, s1, w2, s2) = _weights(e, d, f, 4, 32)
    plan = mld.MoeExperts(e, k, d, f, max_tokens=n)
    x = rng.standard_normal((n, d)).astype(np.float16)
    ids, weights = _ids(rng, n, e, k).astype(np.int32), rng.random((n, k)).astype(np.float32)
    for rows in (n, 1, 16, 17, 2, n, 0):  # 16 tokens are 32 pairs, the most that go the one way
        out = torch.full((n, d), 3.0, dtype=torch.float16, device="cuda")
        plan.run(_dev(x[:rows]), _dev(ids[:rows]), _dev(weights[:rows]), w1, s1, w2, s2, out[:rows])
        got = out.cpu().numpy().astype(np.float64)
        want, size = ref.experts(x[:rows], ids[:rows], weights[:rows], first, second, None, False)
        assert (np.abs(got[:rows] - want) <= _bound(want, size, True)).all() and (got[rows:] == 3).all()
    assert plan.device_status() == 0


def test_two_plans_at_once_on_two_streams(mld):
    e, k, d, f, n = 8, 2, 256, 128, 90
    rng = np.random.default_rng(6)
    (first, second), (w1, s1, w2, s2) = _weights(e, d, f, 4, 32)
    x, ids, weights = rng.standard_normal((n, d)).astype(np.float16), _ids(rng, n, e, k).astype(np.int32), rng.random((n, k)).astype(np.float32)
    xd, idd, wd = _dev(x), _dev(ids), _dev(weights)
    streams = [torch.cuda.Stream() for _ in range(2)]
    plans = [mld.MoeExperts(e, k, d, f, max_tokens=n, force_path=p) for p in (mld.MOE_PATH_FEW_ROWS, mld.MOE_PATH_MANY_ROWS)]
    outs = [torch.empty(20, n, d, dtype=torch.float16, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(20):
        for s, p, o in zip(streams, plans, outs):
            p.run(xd, idd, wd, w1, s1, w2, s2, o[i], stream=s)
    torch.cuda.synchronize()
    want, size = ref.experts(x, ids, weights, first, second, None, False)
    for p, o, many in zip(plans, outs, (False, True)):
        assert p.device_status() == 0 and (o == o[0]).all()
        assert (np.abs(o[0].cpu().numpy().astype(np.float64) - want) <= _bound(want, size, many)).all()


@pytest.mark.parametrize("large", [0.3, 40.0])
def test_scales_whose_multiples_leave_fp16(mld, large):
    """Scales at which the short way from a nibble to a weight is not open, beside some at which it is."""
    e, k, d, f, n = 3, 1, 128, 64, 50
    rng = np.random.default_rng(9)
    (first, second), (w1, s1, w2, s2) = _weights(e, d, f, 4, 32)
    up = np.ones((e, d // 32, 2 * f))
    up[:, 1::2] = large / s1.float().max().item()
    s1 = (s1.double() * torch.from_numpy(up).cuda()).half()
    codes = first / np.repeat(_weights(e, d, f, 4, 32)[1][1].cpu().numpy().astype(np.float64), 32, 1).transpose(0, 2, 1)
    first = np.rint(codes) * np.repeat(s1.cpu().numpy().astype(np.float64), 32, 1).transpose(0, 2, 1)
    x = (rng.standard_normal((n, d)) / (20 * large)).astype(np.float16)
    ids, weights = _ids(rng, n, e, k).astype(np.int32), rng.random((n, k)).astype(np.float32)
    for path in (mld.MOE_PATH_FEW_ROWS, mld.MOE_PATH_MANY_ROWS):
        plan = mld.MoeExperts(e, k, d, f, max_tokens=n, force_path=path)
        out = torch.empty(n, d, dtype=torch.float16, device="cuda")
        plan.run(_dev(x), _dev(ids), _dev(weights), w1, s1, w2, s2, out)
        want, size = ref.experts(x, ids, weights, first, second, None, False)
        assert (np.abs(out.cpu().numpy() - want) <= _bound(want, size, path == mld.MOE_PATH_MANY_ROWS)).all()


@pytest.mark.parametrize("path,n", [("few", 40), ("many", 300)])
@pytest.mark.parametrize("bits", [4, 8])
def test_a_hundred_calls_give_the_same_bits(mld, path, n, bits):
    """More boxes of weights than the rings hold, over and over: nothing is overwritten before it has been read."""
    e, k, d, f = 16, 4, 1024, 512
    rng = np.random.default_rng(n)
    w = [torch.randint(0, 256, (e, 2 * f * d * bits // 8), dtype=torch.uint8, device="cuda"), (0.002 * torch.rand(e, 1, 2 * f, device="cuda")).half(),
         torch.randint(0, 256, (e, f * d * bits // 8), dtype=torch.uint8, device="cuda"), (0.002 * torch.rand(e, 1, d, device="cuda")).half()]
    x, ids, weights = _dev(rng.standard_normal((n, d)).astype(np.float16)), _dev(_ids(rng, n, e, k).astype(np.int32)), _dev(rng.random((n, k)).astype(np.float32))
    plan = mld.MoeExperts(e, k, d, f, weight_bits=bits, block=0, max_tokens=n,
                          force_path=mld.MOE_PATH_FEW_ROWS if path == "few" else mld.MOE_PATH_MANY_ROWS)
    first, out = torch.empty(n, d, dtype=torch.float16, device="cuda"), torch.empty(n, d, dtype=torch.float16, device="cuda")
    plan.run(x, ids, weights, *w, first)
    for _ in range(100):
        plan.run(x, ids, weights, *w, out)
        assert torch.equal(out, first)
