"""Routing of tokens to experts against the definition in 64 bits: the same experts, always."""
import numpy as np
import pytest
import torch

from tests import ffn_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mld():
    import __graft_entry__ as g
    return g.import_package()


def _run(mld, logits, bias, top_k, score, groups, top_groups, best, renormalise, factor):
    n, e = logits.shape
    x = torch.from_numpy(logits).cuda()
    ids, weights = torch.full((n, top_k), 99, dtype=torch.int32, device="cuda"), torch.full((n, top_k), 9.0, device="cuda")
    r = mld.MoeRouter(e, top_k, score=score, groups=groups, top_groups=top_groups, group_best=best, renormalise=renormalise,
                      factor=factor, f16=logits.dtype == np.float16)
    r.run(x, ids, weights, bias=None if bias is None else torch.from_numpy(bias).cuda())
    want_ids, want = ref.route(logits, bias, top_k, score == mld.MOE_SIGMOID, groups, top_groups, best, renormalise, factor)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    got = weights.cpu().numpy()
    # exp to 2 ulp, its argument's rounding (2^-24 times up to 20 between two chosen logits, more for smaller weights), a sum, two divisions
    big = np.abs(want) > 1e-9
    assert np.allclose(got[big], want[big], rtol=1e-5, atol=0) and (np.abs(got - want)[~big] <= 1e-9).all()
    return ids, weights


CASES = [(1, 128, 8, 1, 1, 1), (1, 1, 1, 1, 1, 1), (5, 3, 3, 1, 1, 1), (33, 60, 4, 1, 1, 1), (100, 64, 6, 8, 3, 1), (100, 64, 6, 8, 3, 2),
         (257, 256, 8, 8, 4, 2), (50, 160, 6, 8, 3, 1), (20, 1024, 32, 32, 7, 2), (20, 511, 10, 1, 1, 1), (64, 66, 4, 3, 2, 2),
         (9, 96, 16, 32, 8, 2), (9, 320, 1, 5, 5, 2)]


@pytest.mark.parametrize("n,e,k,groups,top_groups,best", CASES)
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_experts_and_weights(mld, n, e, k, groups, top_groups, best, sigmoid, with_bias, dtype):
    rng = np.random.default_rng(n * e + k)
    logits = (1.5 * rng.standard_normal((n, e)) + 0.5 * rng.standard_normal(e)).astype(dtype)
    bias = (0.2 * rng.standard_normal(e)).astype(np.float32) if with_bias else None
    score = mld.MOE_SIGMOID if sigmoid else mld.MOE_SOFTMAX
    _run(mld, logits, bias, k, score, groups, top_groups, best, True, 1.0)
    _run(mld, logits, bias, k, score, groups, top_groups, best, False, 2.5)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("with_bias", [False, True])
def test_ties_infinities_nan_and_experts_that_run_out(mld, sigmoid, with_bias):
    rng = np.random.default_rng(3)
    score = mld.MOE_SIGMOID if sigmoid else mld.MOE_SOFTMAX
    logits = rng.integers(-2, 3, (40, 48)).astype(np.float32)  # five values among 48 experts
    logits[0] = -np.inf
    logits[1] = np.nan
    logits[2, 3:] = -np.inf
    logits[3, 5], logits[3, 6] = np.nan, -0.0
    logits[4] = np.where(np.arange(48) % 2 == 0, 0.0, -0.0)
    logits[5] += 60  # sigmoids that round to 1
    logits[6] -= 200  # sigmoids that vanish in 32 bits
    logits[7] = np.finfo(np.float32).min
    logits[8, 17] = np.inf
    bias = None
    if with_bias:
        bias = (rng.integers(-1, 2, 48) * 0.25).astype(np.float32)
        bias[9] = -np.inf
    for groups, top_groups, best in ((1, 1, 1), (6, 2, 1), (6, 2, 2), (24, 8, 2)):
        _run(mld, logits, bias, 6, score, groups, top_groups, best, True, 1.0)
    _run(mld, logits[:6], bias, 6, score, 1, 1, 1, False, 1.0)


def test_strided_logits_and_another_stream(mld):
    rng = np.random.default_rng(8)
    wide = torch.from_numpy(rng.standard_normal((77, 200)).astype(np.float16)).cuda()
    logits = wide[:, 3:131]
    ids, weights = torch.empty(77, 8, dtype=torch.int32, device="cuda"), torch.empty(77, 8, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    mld.MoeRouter(128, 8).run(logits, ids, weights, stream=s)
    s.synchronize()
    want, w = ref.route(logits.cpu().numpy(), None, 8, False, 1, 1, 1, True, 1.0)
    assert np.array_equal(ids.cpu().numpy(), want)
    one = wide[:1, :128].expand(5, 128)
    ids, weights = torch.empty(5, 8, dtype=torch.int32, device="cuda"), torch.empty(5, 8, device="cuda")
    mld.MoeRouter(128, 8).run(one, ids, weights)
    assert (ids == ids[0]).all() and (weights == weights[0]).all()
