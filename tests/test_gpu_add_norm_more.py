"""Codes of rows whose values are large against their spread, and of rows at the ends of 32 bits; products on codes with small plans."""
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


def _codes(mld, x, g, offset, symmetric, residual=None):
    n, w = x.shape
    codes, params = torch.full((n, -(-w // 16) * 16), 77, dtype=torch.int8, device="cuda"), torch.empty(n, 3, device="cuda")
    total = torch.empty_like(_dev(x)) if residual is not None else None
    mld.add_rms_norm(_dev(x), weight=None if g is None else _dev(g), residual=None if residual is None else _dev(residual), sum_out=total,
                     codes=codes, params=params, symmetric=symmetric, weight_offset=offset)
    return codes.cpu().numpy()[:, :w], params.cpu().numpy().astype(np.float64)


def _check(mld, x, g, offset, symmetric, residual=None):
    _, v, rstd = ref.add_norm(x, residual, g, 1e-6, offset if g is not None else 0.0)
    q, scale, zero = ref.codes(v, rstd, symmetric)
    got, p = _codes(mld, x, g, offset, symmetric, residual)
    assert np.array_equal(got, q), (got != q).sum()
    # the parameters: as in the norm's own test, 64 roundings of 32 bits at most, the zero point's relative to its largest term
    assert (np.abs(p[:, :1] - scale) <= 64 * U32 * scale).all()
    assert (np.abs(p[:, 1:2] - zero) <= 64 * U32 * (np.abs(zero) + 256 * scale)).all()


@pytest.mark.parametrize("n,w", [(40, 200), (300, 2048), (200, 1155), (30, 8192), (3, 4096)])
@pytest.mark.parametrize("mean,spread", [(100.0, 1.0), (1000.0, 1.0), (-1000.0, 0.01), (3.0e5, 1.0), (1.0e-3, 1.0e-5)])
@pytest.mark.parametrize("offset", [0.0, 1.0])
@pytest.mark.parametrize("symmetric", [True, False])
def test_rows_far_from_zero_in_32_bits(mld, n, w, mean, spread, offset, symmetric):
    """v = h (offset + w) is rounded relative to itself, codes are relative to the row's span."""
    rng = np.random.default_rng(w)
    x = (mean + spread * rng.standard_normal((n, w))).astype(np.float32)
    weights = [((1 - offset) + 1e-6 * rng.standard_normal(w)).astype(np.float32), None if offset == 0 else np.zeros(w, np.float32)]
    for g in weights:
        _check(mld, x, g, offset, symmetric)


@pytest.mark.parametrize("n,w", [(40, 200), (300, 2048), (200, 1155), (30, 8192), (3, 4096)])
@pytest.mark.parametrize("symmetric", [True, False])
def test_rows_far_from_zero_in_16_bits(mld, n, w, symmetric):
    rng = np.random.default_rng(w)
    x = (1000 + 2 * rng.standard_normal((n, w))).astype(np.float16)
    r = rng.standard_normal((n, w)).astype(np.float16)
    _check(mld, x, (0.001 * rng.standard_normal(w)).astype(np.float16), 1.0, symmetric, r)
    _check(mld, np.full((n, w), 1000, np.float16), (0.001 * rng.standard_normal(w)).astype(np.float16), 1.0, symmetric)
    _check(mld, x, (1 + 0.001 * rng.standard_normal(w)).astype(np.float16), 0.0, symmetric, r)


@pytest.mark.parametrize("w", [256, 1155, 4096])
def test_spans_that_leave_32_bits_and_subnormal_ones(mld, w):
    rng = np.random.default_rng(w)
    x = (1e17 * rng.uniform(-1, 1, (5, w))).astype(np.float32)
    x[:, 0], x[:, 1] = 1e17, -1e17
    _check(mld, x, np.full(w, 3.3e21, np.float32), 0.0, False)
    x = (1e-21 * rng.uniform(0.5, 1, (5, w))).astype(np.float32)
    g = (1e-21 * rng.uniform(0.5, 1, w)).astype(np.float32)  # products are subnormal in 32 bits
    _, v, rstd = ref.add_norm(x, None, g, 1e-6, 0.0)
    for symmetric in (True, False):
        assert np.array_equal(_codes(mld, x, g, 0.0, symmetric)[0], ref.codes(v, rstd, symmetric)[0])


@pytest.mark.parametrize("most", [1, 4, 8, 16])
@pytest.mark.parametrize("symmetric", [True, False])
def test_products_on_codes_with_plans_of_few_tokens(mld, most, symmetric):
    """A plan whose calls with fp16 activations all take the decode kernel serves codes, too."""
    n, k = 264, 272
    rng = np.random.default_rng(most)
    wq = rng.integers(-128, 128, (n, k))
    packed, sums = mld.pack_weights(_dev(wq.astype(np.int8)), (n, 1, 1, k), 8, want_sum=True)
    scale = np.exp(0.3 * rng.standard_normal(n)).astype(np.float16)
    for cached in (False, True):
        plan = mld.FullyConnectedPlan(n, k, 8, max_tokens=most, src_layout=mld.LAYOUT_ROW_MAJOR, dst_layout=mld.LAYOUT_ROW_MAJOR,
                                      prefill_act_quant=1 if symmetric else 2, cache_prepared_weights=cached)
        plan.set_weights_sum(sums)
        for tokens in {1, most}:
            q = rng.integers(-128, 128, (tokens, k))
            p = np.stack((rng.uniform(0.001, 0.002, tokens), np.zeros(tokens) if symmetric else rng.uniform(-0.1, 0.1, tokens), np.zeros(tokens)), 1)
            p = p.astype(np.float32)
            y = torch.empty(tokens, n, dtype=torch.float16, device="cuda")
            plan.run_codes(_dev(q.astype(np.int8)), _dev(p), packed, _dev(scale), y, tokens)
            p, s = p.astype(np.float64), scale.astype(np.float64)
            want = (q @ wq.T * p[:, :1] + p[:, 1:2] * wq.sum(1)) * s
            # exact sums of integers; four products and an addition in 32 bits, one rounding to fp16
            size = (np.abs(q @ wq.T) * p[:, :1] + np.abs(p[:, 1:2] * wq.sum(1))) * s
            bound = 8 * U32 * size + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
            assert (np.abs(y.cpu().numpy() - want) <= bound).all()
        assert plan.device_status() == 0


@pytest.mark.parametrize("tokens,k,n", [(1, 256, 64), (77, 272, 568), (130, 1040, 262), (513, 512, 1024)])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("route", ["tensor memory", "shared memory", "prepared"])
@pytest.mark.parametrize("row_major", [True, False])
def test_outputs_are_rounded_once(mld, tokens, k, n, symmetric, route, row_major):
    rng = np.random.default_rng(tokens + k)
    wq = rng.integers(-128, 128, (n, k))
    packed, sums = mld.pack_weights(_dev(wq.astype(np.int8)), (n, 1, 1, k), 8, want_sum=True)
    n4 = (n + 3) // 4 * 4
    scale, bias = np.zeros(n4, np.float16), np.zeros(n4, np.float16)
    scale[:n], bias[:n] = np.exp(0.3 * rng.standard_normal(n)) / (70 * np.sqrt(k)), rng.standard_normal(n)
    plan = mld.FullyConnectedPlan(n, k, 8, has_bias=True, max_tokens=tokens, src_layout=mld.LAYOUT_ROW_MAJOR, force_path=mld.PATH_GEMM,
                                  dst_layout=mld.LAYOUT_ROW_MAJOR if row_major else mld.LAYOUT_SLICED, prefill_act_quant=1 if symmetric else 2,
                                  cache_prepared_weights=route == "prepared", prefill_route=dict(zip(("tensor memory", "prepared", "shared memory"), (1, 0, 3)))[route])
    plan.set_weights_sum(sums)
    q = rng.integers(-128, 128, (tokens, (k + 15) // 16 * 16))
    q[:, k:] = 0
    p = np.stack((rng.uniform(0.01, 0.02, tokens), np.zeros(tokens) if symmetric else rng.uniform(-1, 1, tokens), np.zeros(tokens)), 1).astype(np.float32)
    y = torch.full((tokens, n) if row_major else (n4 // 4, tokens, 4), 9.0, dtype=torch.float16, device="cuda")
    plan.run_codes(_dev(q.astype(np.int8)), _dev(p), packed, _dev(scale), y, tokens, bias=_dev(bias))
    assert plan.device_status() == 0
    got = y.cpu().numpy().astype(np.float64) if row_major else y.cpu().numpy().astype(np.float64).transpose(1, 0, 2).reshape(tokens, n4)[:, :n]
    s, b, p = scale[:n].astype(np.float64), bias[:n].astype(np.float64), p.astype(np.float64)
    product, zero = q[:, :k] @ wq.T * p[:, :1] * s, p[:, 1:2] * wq.sum(1) * s
    want = product + zero + b
    # exact sums of integers below 2^24; at most six roundings of 32 bits of each term (the sums as 32-bit numbers, products, additions),
    # and one to fp16
    bound = 6 * U32 * (np.abs(product) + np.abs(zero) + np.abs(b)) + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
    assert (np.abs(got - want) <= bound).all(), np.max(np.abs(got - want) / bound)
