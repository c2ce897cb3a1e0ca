"""Routing where values of groups tie or nearly do: the same groups as in 64 bits."""
import numpy as np
import pytest
import torch

from tests import ffn_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mld():
    import __graft_entry__ as g
    return g.import_package()


def _ids(mld, logits, bias, top_k, score, groups, top_groups, best):
    n, e = logits.shape
    ids, weights = torch.full((n, top_k), 99, dtype=torch.int32, device="cuda"), torch.empty(n, top_k, device="cuda")
    r = mld.MoeRouter(e, top_k, score=score, groups=groups, top_groups=top_groups, group_best=best, f16=logits.dtype == np.float16)
    r.run(torch.from_numpy(logits).cuda(), ids, weights, bias=None if bias is None else torch.from_numpy(bias).cuda())
    want, gates = ref.route(logits, bias, top_k, score == mld.MOE_SIGMOID, groups, top_groups, best, True, 1.0)
    assert np.array_equal(ids.cpu().numpy(), want), (ids.cpu().numpy() != want).any(1).sum()
    assert np.allclose(weights.cpu().numpy(), gates, rtol=1e-5, atol=1e-30)
    return want


def test_groups_whose_best_values_are_equal_though_their_logits_are_not(mld):
    """Sigmoids of 40 and 50 are 1 in 64 bits, and of equal groups the first is kept: with a bias of zeros, and without one."""
    logits = np.full((1, 8), -3, np.float32)
    logits[0, 1], logits[0, 6] = 40, 50
    for bias in (None, np.zeros(8, np.float32)):
        assert _ids(mld, logits, bias, 1, mld.MOE_SIGMOID, 2, 1, 1)[0, 0] == 1


@pytest.mark.parametrize("e,groups", [(64, 8), (60, 6), (512, 32), (96, 32)])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("values", ["large", "small", "vanishing", "near zero", "close", "ties", "ordinary"])
def test_groups_without_a_bias(mld, e, groups, dtype, sigmoid, values):
    rng = np.random.default_rng(e)
    n = 64
    x = rng.standard_normal((n, e))
    if values == "large":
        x = 40 + 12 * x
    elif values == "small":
        x = -40 - 12 * np.abs(x)
    elif values == "vanishing":  # one expert far above the others, whose exponentials vanish
        x = x * 30 - (800 if dtype is np.float32 else 900)
        x[:, 5] = 10
    elif values == "near zero":
        x = x * (1e-18 if dtype is np.float32 else 1e-7)
    elif values == "close":
        x = 1 + x * 1e-6
    elif values == "ties":
        x = np.round(2 * x)
    score = mld.MOE_SIGMOID if sigmoid else mld.MOE_SOFTMAX
    for top_groups in (1, 2, groups - 1):
        _ids(mld, x.astype(dtype), None, min(4, top_groups * (e // groups)), score, groups, top_groups, 1)


@pytest.mark.parametrize("large", [50.0, 5000.0, 3.0e7])
def test_sums_of_two_values_of_opposite_signs(mld, large):
    """A group's sum is small, its terms are not: it is as exact as those, not as itself."""
    rng = np.random.default_rng(4)
    n, e, groups = 500, 32, 4
    spread = 30 * large * 2.0 ** -24
    logits = (spread * rng.standard_normal((n, e))).astype(np.float32)
    bias = np.full(e, -large, np.float32)
    bias[np.arange(groups) * (e // groups) + [3, 0, 7, 5]] = large
    _ids(mld, logits, bias, 1, mld.MOE_SIGMOID, groups, 1, 2)
    _ids(mld, logits, bias, 1, mld.MOE_SOFTMAX, groups, 1, 2)
