"""Experts' networks where a block has many items, and at the limits of their plans."""
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


def _few_matrices(seed, d, f, bits, block, experts, distinct):
    """`distinct` experts' matrices in 64 bits, and those of `experts` that take them in turn on the device."""
    rng = np.random.default_rng(seed)
    host, dev = [], []
    for o, i in ((2 * f, d), (d, f)):
        ms = [ref.matrix(rng, o, i, bits, block) for _ in range(distinct)]
        host.append(np.stack([m[2] for m in ms]))
        for part in range(2):
            one = _dev(np.stack([m[part] for m in ms]))
            dev.append(one[torch.arange(experts, device="cuda") % distinct].contiguous())
    return host, dev


@pytest.mark.parametrize("d,f", [(4096, 128), (128, 4096), (4096, 96)])
@pytest.mark.parametrize("bits,block", [(4, 32), (8, 0)])
def test_items_of_one_box_and_many_of_them(mld, d, f, bits, block):
    """A hundred items to a block, each a single box of weights: rows are those of the item, over and over."""
    e, k, n, distinct = 256, 4, 128, 4
    (first, second), w = _few_matrices(d + f, d, f, bits, block, e, distinct)
    rng = np.random.default_rng(f)
    x, gates = rng.standard_normal((n, d)).astype(np.float16), rng.random((n, k)).astype(np.float32)
    ids = np.argsort(rng.random((n, e)), 1)[:, :k].astype(np.int32)
    plan = mld.MoeExperts(e, k, d, f, weight_bits=bits, block=block, max_tokens=n, force_path=mld.MOE_PATH_FEW_ROWS)
    xd, idd, gd = _dev(x), _dev(ids), _dev(gates)
    start, out = torch.empty(n, d, dtype=torch.float16, device="cuda"), torch.empty(n, d, dtype=torch.float16, device="cuda")
    plan.run(xd, idd, gd, *w, start)
    for _ in range(50):
        plan.run(xd, idd, gd, *w, out)
        assert torch.equal(out, start)
    assert plan.device_status() == 0
    want, size = ref.experts(x, ids % distinct, gates, first, second, None, False)
    bound = ref.experts_bound(want, size, False)
    got = out.cpu().numpy().astype(np.float64)
    assert (np.abs(got - want) <= bound).all(), np.max(np.abs(got - want) / bound)


def test_a_plan_that_does_not_fit_leaves_no_error_behind(mld):
    with pytest.raises(mld.MldError, match="experts' workspace"):
        mld.MoeExperts(1024, 32, 32768, 32768, max_tokens=65536)  # 270 GB
    logits = torch.zeros(3, 64, dtype=torch.float16, device="cuda")
    ids, weights = torch.empty(3, 2, dtype=torch.int32, device="cuda"), torch.empty(3, 2, device="cuda")
    mld.MoeRouter(64, 2).run(logits, ids, weights)
    assert (ids.cpu() == torch.tensor([0, 1])).all()
