"""Edges of the 4-bit cache's operators: values that are not finite, sizes near 2^31, batches of very uneven sequences.

Tolerances are those of the operators' other tests: attention 2^-11 of the output and of sum(p |v|), a tenth on top; rotation a
handful of roundings of 2^-24 of a row's size and of the output's type."""
import numpy as np
import pytest
import torch

from tests import kv4_ref as ref
from tests.test_gpu_kv4 import _attention_case, _dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mld():
    import __graft_entry__ as g
    return g.import_package()


@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_small_values_beside_nan_that_a_row_does_not_see(mld, head_dim):
    """A window that has left a NaN behind: the rows after it are as exact as without it."""
    rng = np.random.default_rng(head_dim)
    n, m, window, page = 400, 48, 12, 16
    cache = mld.Kv4Cache(1, head_dim, page, n // page)
    k = rng.standard_normal((n, 1, head_dim)).astype(np.float16)
    v = (3e-4 * rng.standard_normal((n, 1, head_dim))).astype(np.float16)
    lost = np.arange(n - m - 4, n, 16)  # every block of rows has one in what its first rows see
    v[lost, 0, 5] = np.nan
    cache.write(_dev(k), _dev(v), torch.arange(n, dtype=torch.int32, device="cuda"))
    q = (6 * rng.standard_normal((m, 1, head_dim))).astype(np.float16)
    at = np.arange(n - m, n)[:, None]
    sees = ((lost <= at) & (lost > at - window)).any(1)
    nan = np.zeros((m, 1, head_dim), bool)
    nan[sees, 0, :32] = True
    assert 4 < sees.sum() < m - 4
    want, size = ref.attention(q, ref.quantise(k), np.nan_to_num(ref.quantise(v)), m, head_dim ** -0.5, window)
    table = torch.arange(n // page, dtype=torch.int32, device="cuda")[None].contiguous()
    for path in (mld.KV4_PATH_FEW_ROWS, mld.KV4_PATH_MANY_ROWS):
        out = torch.zeros(m, 1, head_dim, dtype=torch.float16, device="cuda")
        mld.Kv4Attention(cache, 1, 1, n // page, window=window, force_path=path).run(
            _dev(q), table, _dev(np.int32([n])), out, q_starts=_dev(np.int32([0, m])), max_queries=m)
        got = out.cpu().numpy().astype(np.float64)
        assert np.array_equal(np.isnan(got), nan), path
        tol = 1.1 * 2.0 ** -11 * (np.abs(want) + size) + 2.0 ** -25
        worst = (np.abs(got - want) / tol)[~nan].max()
        assert worst <= 1, (path, worst)
