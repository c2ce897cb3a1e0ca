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


@pytest.mark.parametrize("path", ["few", "many"])
@pytest.mark.parametrize("n", [1, 5, 70])
def test_scales_of_256_inputs(mld, n, path):
    e, k, d, f = 4, 2, 512, 256
    (first, second), w = _few_matrices(7, d, f, 4, 256, e, e)
    rng = np.random.default_rng(n)
    x, gates = rng.standard_normal((n, d)).astype(np.float16), rng.random((n, k)).astype(np.float32)
    ids = np.argsort(rng.random((n, e)), 1)[:, :k].astype(np.int32)
    plan = mld.MoeExperts(e, k, d, f, block=256, max_tokens=n, force_path=mld.MOE_PATH_FEW_ROWS if path == "few" else mld.MOE_PATH_MANY_ROWS)
    out = torch.empty(n, d, dtype=torch.float16, device="cuda")
    plan.run(_dev(x), _dev(ids), _dev(gates), *w, out)
    want, size = ref.experts(x, ids, gates, first, second, None, False)
    assert (np.abs(out.cpu().numpy() - want) <= ref.experts_bound(want, size, path == "many")).all()
    assert plan.device_status() == 0


def test_a_call_goes_the_way_that_its_rows_to_an_expert_say(mld):
    """Up to eight rows to an expert, on average, as a plan for few rows; more, as one for many: the same bits."""
    e, k, d, f, n = 4, 2, 512, 256, 60
    (first, second), w = _few_matrices(8, d, f, 4, 32, e, e)
    rng = np.random.default_rng(3)
    x, gates = _dev(rng.standard_normal((n, d)).astype(np.float16)), _dev(rng.random((n, k)).astype(np.float32))
    ids = _dev(np.argsort(rng.random((n, e)), 1)[:, :k].astype(np.int32))
    auto, few, many = (mld.MoeExperts(e, k, d, f, max_tokens=n, force_path=p) for p in (0, mld.MOE_PATH_FEW_ROWS, mld.MOE_PATH_MANY_ROWS))
    for rows in (1, 2, 15, 16, 17, 40, n):
        outs = []
        for plan in (auto, few, many):
            outs.append(torch.empty(rows, d, dtype=torch.float16, device="cuda"))
            plan.run(x[:rows], ids[:rows], gates[:rows], *w, outs[-1])
        assert not torch.equal(outs[1], outs[2])  # (weights in 16 bits, and in their codes)
        assert torch.equal(outs[0], outs[2 if rows * k > 8 * e else 1])


def test_a_plan_that_does_not_fit_leaves_no_error_behind(mld):
    with pytest.raises(mld.MldError, match="experts' workspace"):
        mld.MoeExperts(1024, 32, 32768, 32768, max_tokens=65536)  # 270 GB
    logits = torch.zeros(3, 64, dtype=torch.float16, device="cuda")
    ids, weights = torch.empty(3, 2, dtype=torch.int32, device="cuda"), torch.empty(3, 2, device="cuda")
    mld.MoeRouter(64, 2).run(logits, ids, weights)
    assert (ids.cpu() == torch.tensor([0, 1])).all()


@pytest.mark.parametrize("path", ["few", "many"])
@pytest.mark.parametrize("n", [1, 40, 300])
@pytest.mark.parametrize("large", [1.0, 3.0e4])
def test_outputs_of_experts_that_leave_16_bits_ahead_of_their_weights(mld, n, path, large):
    """Experts' outputs of a few hundred thousands, weights that bring the sums back: the same range, however many tokens come along."""
    e, k, d, f = 4, 2, 256, 128
    (first, second), (w1, s1, w2, s2) = _few_matrices(9, d, f, 4, 32, e, e)
    s2 = (s2.double() * large).half()
    second = np.rint(second / _spread(_few_matrices(9, d, f, 4, 32, e, e)[1][3], f)) * _spread(s2, f)
    rng = np.random.default_rng(n)
    x, gates = rng.standard_normal((n, d)).astype(np.float16), (rng.random((n, k)) / large).astype(np.float32)
    gates[:, 0] *= -1
    gates[0] = 0
    ids = np.argsort(rng.random((n, e)), 1)[:, :k].astype(np.int32)
    res = rng.standard_normal((n, d)).astype(np.float16)
    plan = mld.MoeExperts(e, k, d, f, max_tokens=n, force_path=mld.MOE_PATH_FEW_ROWS if path == "few" else mld.MOE_PATH_MANY_ROWS)
    out = torch.empty(n, d, dtype=torch.float16, device="cuda")
    plan.run(_dev(x), _dev(ids), _dev(gates), w1, s1, w2, s2, out, residual=_dev(res))
    want, size = ref.experts(x, ids, gates, first, second, res, False)
    got = out.cpu().numpy().astype(np.float64)
    bound = ref.experts_bound(want, size, path == "many")
    assert (np.abs(got - want) <= bound).all(), np.max(np.abs(got - want) / bound)
    assert np.array_equal(got[0], res[0])


def _spread(scales, inputs):
    """Scales [experts][groups][outputs] for each of the inputs, [experts][outputs][inputs]."""
    s = scales.double().cpu().numpy()
    return np.repeat(s, inputs // s.shape[1], 1).transpose(0, 2, 1)


@pytest.mark.parametrize("path", ["few", "many"])
@pytest.mark.parametrize("n", [1, 40, 300, 700])
@pytest.mark.parametrize("bits,d,f", [(8, 96, 352), (8, 512, 256), (4, 256, 128)])
@pytest.mark.parametrize("large", [1.0, 200.0])
def test_weights_with_a_scale_to_an_output_are_not_rounded(mld, n, path, bits, d, f, large):
    """Both kernels within the errors of gated values and results alone; experts' outputs may leave 16 bits ahead of their weights."""
    e, k = 5, 2
    (first, second), (w1, s1, w2, s2) = _few_matrices(d + bits, d, f, bits, 0, e, e)
    s2, old = (s2.double() * large).half(), _spread(s2, f)
    second = np.rint(second / old) * _spread(s2, f)
    rng = np.random.default_rng(n)
    x, gates = (30 * rng.standard_normal((n, d))).astype(np.float16), (rng.random((n, k)) / (900 * large)).astype(np.float32)
    ids = np.argsort(rng.random((n, e)), 1)[:, :k].astype(np.int32)
    ids[3::11, 1] = -1
    plan = mld.MoeExperts(e, k, d, f, weight_bits=bits, block=0, max_tokens=n, activation=n % 2, force_path=mld.MOE_PATH_FEW_ROWS if path == "few" else mld.MOE_PATH_MANY_ROWS)
    out = torch.empty(n, d, dtype=torch.float16, device="cuda")
    plan.run(_dev(x), _dev(ids), _dev(gates), w1, s1, w2, s2, out)
    want, size = ref.experts(x, ids, gates, first, second, None, n % 2 == 1)
    got = out.cpu().numpy().astype(np.float64)
    bound = ref.experts_bound(want, size, False)
    assert (np.abs(got - want) <= bound).all(), np.max(np.abs(got - want) / bound)
    assert plan.device_status() == 0
    signal = np.sqrt((want ** 2).sum())
    # two roundings to 16 bits, of at most 2^-11 each, uncorrelated; sums in 32 bits are far below
    assert np.sqrt(((got - want) ** 2).sum()) <= 2.0 ** -11 * np.sqrt(2) / np.sqrt(3) * 1.05 * signal
