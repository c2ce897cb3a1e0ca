"""Residual and RMS norm with an output in 8 bits, and products on its codes, against the formulas in 64 bits."""
import numpy as np
import pytest
import torch

from tests import ffn_ref as ref

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24


@pytest.fixture(scope="module")
def mld():
    import __graft_entry__ as g
    return g.import_package()


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _make(rng, n, w, dtype, offset):
    x = rng.standard_normal((n, w)).astype(dtype)
    r = (rng.standard_normal((n, w)) * np.exp(0.8 * rng.standard_normal(w))).astype(dtype)
    g = ((1 - offset) + 0.2 * rng.standard_normal(w)).astype(dtype)
    return x, r, g


def _check_out(got, want, dtype):
    # 32 bits: the sum of squares (two roundings a value at most on average, of positive terms: a relative error below
    # width / 32 / 8 + 12 roundings of partial sums, halved by the root), three products, an addition, a division and a root
    bound = (np.finfo(dtype).eps / 2 + 64 * U32) * np.abs(want) + 2.0 ** -25
    assert (np.abs(got - want) <= bound).all(), np.max(np.abs(got - want) - bound)


@pytest.mark.parametrize("n,w", [(1, 4096), (1, 1), (3, 8), (5, 31), (2, 32), (7, 250), (149, 256), (300, 1024), (333, 1155), (3, 1032),
                                 (40, 2048), (700, 4096), (9, 5003), (150, 8192), (2, 16384), (150, 16377)])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("symmetric,offset", [(True, 0.0), (False, 1.0)])
def test_sum_norm_and_codes(mld, n, w, dtype, symmetric, offset):
    rng = np.random.default_rng(n * w)
    x, r, g = _make(rng, n, w, dtype, offset)
    h, v, rstd = ref.add_norm(x, r, g, 1e-6, offset)
    q, scale, zero = ref.codes(v, rstd, symmetric)
    wq = -(-w // 16) * 16
    xd, rd, gd = _dev(x), _dev(r), _dev(g)
    total, y = torch.empty_like(xd), torch.empty_like(xd)
    codes, params = torch.full((n, wq), 77, dtype=torch.int8, device="cuda"), torch.empty(n, 3, device="cuda")
    mld.add_rms_norm(xd, weight=gd, residual=rd, sum_out=total, out=y, codes=codes, params=params, symmetric=symmetric, weight_offset=offset)
    torch.cuda.synchronize()
    assert np.array_equal(total.cpu().numpy(), h)
    _check_out(y.cpu().numpy().astype(np.float64), v * rstd, dtype)
    got = codes.cpu().numpy()
    assert np.array_equal(got[:, :w], q) and not got[:, w:].any()
    p = params.cpu().numpy().astype(np.float64)
    assert (np.abs(p[:, :1] - scale) <= 64 * U32 * scale).all()
    assert (np.abs(p[:, 1:2] - zero) <= 64 * U32 * (np.abs(zero) + 256 * scale)).all() and not p[:, 2].any()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("w", [512, 2048, 2047])
def test_in_place_strides_and_missing_parts(mld, dtype, w):
    rng = np.random.default_rng(w)
    n = 200
    x, r, g = _make(rng, n, w, dtype, 0.0)
    wide = torch.zeros(n, w + 24, dtype=torch.float16 if dtype is np.float16 else torch.float32, device="cuda")
    stream = wide[:, 8:8 + w]  # the residual stream inside a larger tensor, updated in place
    stream.copy_(_dev(r))
    h, v, rstd = ref.add_norm(x, r, g, 1e-5, 0.0)
    y, xd = torch.empty(n, w, dtype=wide.dtype, device="cuda"), _dev(x)
    mld.add_rms_norm(xd, weight=_dev(g), residual=stream, sum_out=stream, out=xd, eps=1e-5)  # y over x
    assert np.array_equal(stream.cpu().numpy(), h) and not wide[:, :8].any() and not wide[:, 8 + w:].any()
    _check_out(xd.cpu().numpy().astype(np.float64), v * rstd, dtype)
    # no residual, no weight, codes alone; out over x beside codes that are worked out again
    h, v, rstd = ref.add_norm(x, None, None, 1e-5, 0.0)
    wq = -(-w // 16) * 16
    codes, params, xd = torch.empty(n, wq, dtype=torch.int8, device="cuda"), torch.empty(n, 3, device="cuda"), _dev(x)
    mld.add_rms_norm(xd, codes=codes, params=params, eps=1e-5, symmetric=False, out=xd)
    assert np.array_equal(codes.cpu().numpy()[:, :w], ref.codes(v, rstd, False)[0])
    _check_out(xd.cpu().numpy().astype(np.float64), v * rstd, dtype)
    # one row of the input for all tokens
    one = _dev(x[:1]).expand(n, w)
    mld.add_rms_norm(one, out=y, eps=1e-5)
    assert (y == y[0]).all()
    mld.add_rms_norm(one, residual=_dev(r), out=y, eps=1e-5)  # the sum is not wanted
    h, v, rstd = ref.add_norm(np.repeat(x[:1], n, 0), r, None, 1e-5, 0.0)
    _check_out(y.cpu().numpy().astype(np.float64), v * rstd, dtype)


def test_values_on_borders_between_codes(mld):
    """Multiples of half a step: every second value lies on a border, and goes up."""
    w = 512
    for dtype in (np.float16, np.float32):
        x = np.tile((np.arange(w) - 254).astype(dtype) / 2, (3, 1))  # -127 .. 127 and beyond, in halves
        x[:, -3:] = 127, -127, 0.5
        h, v, rstd = ref.add_norm(x, None, None, 1e-6, 0.0)
        codes, params = torch.empty(3, w, dtype=torch.int8, device="cuda"), torch.empty(3, 3, device="cuda")
        for symmetric in (True, False):
            mld.add_rms_norm(_dev(x), codes=codes, params=params, symmetric=symmetric)
            want = ref.codes(v, rstd, symmetric)[0]
            assert np.array_equal(codes.cpu().numpy(), want)


def test_rows_of_zeros_equal_values_tiny_values_infinities_and_nan(mld):
    w = 1030
    x = np.random.default_rng(5).standard_normal((8, w)).astype(np.float32)
    x[0] = 0
    x[1] = 2.5
    x[2] *= 1e-30
    x[3] *= 1e-42  # subnormal
    x[4, 77] = np.inf
    x[5, 1029] = np.nan
    x[6] *= 1e25   # squares leave 32 bits
    codes, params = torch.empty(8, 1040, dtype=torch.int8, device="cuda"), torch.empty(8, 3, device="cuda")
    y = torch.empty(8, w, device="cuda")
    for symmetric in (True, False):
        mld.add_rms_norm(_dev(x), out=y, codes=codes, params=params, eps=1e-6, symmetric=symmetric)
        h, v, rstd = ref.add_norm(x[[0, 1, 2, 3, 7]], None, None, 1e-6, 0.0)
        q, scale, zero = ref.codes(v, rstd, symmetric)
        got, p = codes.cpu().numpy(), params.cpu().numpy()
        assert np.array_equal(got[[0, 1, 2, 3, 7], :w], q)
        ok = [0, 1, 2, 7]  # (the subnormal row's scale is below 32 bits' normal range)
        assert np.allclose(p[ok, 0], scale[[0, 1, 2, 4], 0], rtol=1e-5, atol=0)
        assert np.isnan(p[4:7, :2]).all() and not got[4:7].any() and np.isfinite(p[[0, 1, 2, 3, 7]]).all()
        out = y.cpu().numpy()
        assert np.isnan(out[4, 77]) and np.isnan(out[5]).all() and not out[0].any()


@pytest.mark.parametrize("tokens,k,n", [(1, 256, 64), (17, 2048, 4096), (77, 272, 568), (130, 1040, 264), (513, 512, 1024)])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("route", ["auto", "cached"])
def test_product_on_codes_is_the_product_of_the_values(mld, tokens, k, n, symmetric, route):
    rng = np.random.default_rng(tokens + k)
    x, r, g = _make(rng, tokens, k, np.float16, 0.0)
    wq = np.clip(np.rint(rng.standard_normal((n, k)) * 40), -128, 127)
    packed, sums = mld.pack_weights(_dev(wq.astype(np.int8)), (n, 1, 1, k), 8, want_sum=True)
    scale = (np.exp(0.3 * rng.standard_normal(n)) / (40 * np.sqrt(k))).astype(np.float16)
    bias = rng.standard_normal(n).astype(np.float16)
    codes, params = torch.empty(tokens, -(-k // 16) * 16, dtype=torch.int8, device="cuda"), torch.empty(tokens, 3, device="cuda")
    total, y = torch.empty(tokens, k, dtype=torch.float16, device="cuda"), torch.empty(tokens, n, dtype=torch.float16, device="cuda")
    plan = mld.FullyConnectedPlan(n, k, 8, has_bias=True, max_tokens=max(tokens, 20), src_layout=mld.LAYOUT_ROW_MAJOR,
                                  dst_layout=mld.LAYOUT_ROW_MAJOR, prefill_act_quant=1 if symmetric else 2,
                                  cache_prepared_weights=route == "cached", prefill_route=0)
    plan.set_weights_sum(sums)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):  # as a captured step, replayed
        def step():
            mld.add_rms_norm(_dev_x, weight=_dev_g, residual=_dev_r, sum_out=total, codes=codes, params=params, symmetric=symmetric)
            plan.run_codes(codes, params, packed, _dev_s, y, tokens, bias=_dev_b)
        _dev_x, _dev_r, _dev_g, _dev_s, _dev_b = _dev(x), _dev(r), _dev(g), _dev(scale), _dev(bias)
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step()
        y.zero_()
        graph.replay()
        graph.replay()
    torch.cuda.synchronize()
    assert plan.device_status() == 0
    h, v, rstd = ref.add_norm(x, r, g, 1e-6, 0.0)
    q, step_, zero = ref.codes(v, rstd, symmetric)
    a = q * step_ + zero
    w = wq * scale.astype(np.float64)[:, None]
    want = a @ w.T + bias.astype(np.float64)
    # the integers' sums are exact; the parameters' error (64 roundings at most, see above) and the epilogue's four roundings
    # act on both terms; the product is rounded to fp16 ahead of the bias, and again behind it
    size = np.abs((q * step_) @ w.T) + np.abs(zero) * np.abs(w.sum(1)) + 256 * step_ * np.abs(w.sum(1))
    bound = 80 * U32 * size + 2.0 ** -11 * (np.abs(want - bias.astype(np.float64)) + np.abs(want)) * 1.001 + 2.0 ** -23
    got = y.cpu().numpy().astype(np.float64)
    assert (np.abs(got - want) <= bound).all(), np.max(np.abs(got - want) / bound)
