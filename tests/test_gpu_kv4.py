"""Operators around the 4-bit key/value cache, through the C ABI, against plain restatements in 64 bits.

Tolerances.  Attention: the output is rounded to fp16 (2^-11 of it), and so is every weight before the product with the values
(2^-11 of sum(p |v|)); the rest is 32-bit arithmetic (exponentials good to 2^-20 or better, sums), for which a tenth of these
is allowed.  Norm and rotation: 32-bit arithmetic, a handful of roundings of 2^-24 of a pair's size, and of the output's type.
What is held in 4 bits is compared for equality."""
import ctypes

import numpy as np
import pytest
import torch

from tests import kv4_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mld():
    import __graft_entry__ as g
    return g.import_package()


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _slots(rng, tokens, page, pages):
    """A slot for each token, in pages of a random order."""
    order = rng.permutation(pages)[:-(-tokens // page)]
    return (order[np.arange(tokens) // page] * page + np.arange(tokens) % page).astype(np.int32)


# ------------------------------------------------------------------------------------------------- write and read
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("kv_heads,page,tokens,f16", [(1, 16, 1, True), (3, 48, 77, True), (8, 64, 200, False), (5, 128, 33, True)])
def test_write_then_read_gives_the_rounded_values(mld, head_dim, kv_heads, page, tokens, f16):
    rng = np.random.default_rng(head_dim + tokens)
    dt = np.float16 if f16 else np.float32
    k, v = (rng.standard_normal((tokens, kv_heads, head_dim)).astype(dt) * dt(s) for s in (1, 30))
    k[0, 0, :32] = 0                 # a group of zeros
    v[-1, -1, 5] = 60000             # far beside the others
    k[tokens // 2, 0, -32:] *= dt(1e-7) if f16 else dt(1e-7)
    pages = -(-tokens // page) + 2
    slots = _slots(rng, tokens, page, pages)
    cache = mld.Kv4Cache(kv_heads, head_dim, page, pages)
    cache.pool.fill_(0xAB)
    cache.write(_dev(k), _dev(v), _dev(slots))
    gk, gv = (torch.full((tokens, kv_heads, head_dim), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2))
    cache.read(_dev(slots), gk, gv)
    assert np.array_equal(gk.cpu().numpy().astype(np.float64), ref.quantise(k))
    assert np.array_equal(gv.cpu().numpy().astype(np.float64), ref.quantise(v))


def test_a_token_leaves_its_neighbours_alone_and_slots_outside_are_passed_over(mld):
    rng = np.random.default_rng(3)
    cache = mld.Kv4Cache(2, 128, 32, 3, layers=2)
    k = _dev(rng.standard_normal((96, 2, 128)).astype(np.float16))
    every = torch.arange(96, dtype=torch.int32, device="cuda")
    cache.write(k, k * 2, every, layer=1)
    before = cache.pool.clone()
    assert int(before[0].count_nonzero()) == 0
    slots = _dev(np.int32([-1, 37, 96, 2**31 - 1, -2**31]))
    new = _dev(rng.standard_normal((5, 2, 128)).astype(np.float16))
    cache.write(new, -new, slots, layer=1)
    gk, gv = (torch.empty(96, 2, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    cache.read(every, gk, gv, layer=1)
    wk, wv = k.clone(), k * 2
    wk[37], wv[37] = new[1], -new[1]
    assert np.array_equal(gk.cpu().numpy().astype(np.float64), ref.quantise(wk.cpu().numpy()))
    assert np.array_equal(gv.cpu().numpy().astype(np.float64), ref.quantise(wv.cpu().numpy()))
    gk5, gv5 = (torch.full((5, 2, 128), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2))
    cache.read(slots, gk5, gv5, layer=1)
    assert int(gk5[[0, 2, 3, 4]].count_nonzero()) == 0 and int(gv5[[0, 2, 3, 4]].count_nonzero()) == 0
    assert int((cache.pool[0] != before[0]).sum()) == 0


def test_infinities_and_nan_make_their_group_nan_and_no_other(mld):
    k = np.ones((3, 1, 64), np.float16)
    k[0, 0, 3], k[1, 0, 40], k[2, 0, 63] = np.inf, np.nan, -np.inf
    cache = mld.Kv4Cache(1, 64, 16, 1)
    slots = _dev(np.int32([0, 1, 2]))
    cache.write(_dev(k), _dev(k), slots)
    gk, gv = (torch.empty(3, 1, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    cache.read(slots, gk, gv)
    want = ref.quantise(k)
    assert np.isnan(want).sum() == 96
    assert np.array_equal(gk.cpu().numpy().astype(np.float64), want, equal_nan=True)
    assert np.array_equal(gv.cpu().numpy().astype(np.float64), want, equal_nan=True)


# ------------------------------------------------------------------------------------------------ norm and rotation
ROPE = [  # tokens, heads, kv_heads, head_dim, rotary, neighbours, sections, f16
    (1, 32, 8, 128, 128, False, [64], True),
    (3, 4, 4, 64, 64, True, [32], True),
    (77, 7, 1, 256, 64, False, [32], False),
    (130, 5, 5, 64, 16, False, [8], True),
    (9, 16, 2, 128, 96, True, [24, 12, 12], False),
    (33, 3, 3, 128, 128, False, [16, 24, 24], True),
    (5, 2, 1, 256, 256, False, [32, 32, 32, 32], False),
    (4, 2, 2, 64, 0, False, [0], True),
]


@pytest.mark.parametrize("tokens,heads,kv_heads,head_dim,rotary,neighbours,sections,f16", ROPE)
@pytest.mark.parametrize("far", [0, 1 << 17, (1 << 31) - 200])
def test_norm_and_rotation(mld, tokens, heads, kv_heads, head_dim, rotary, neighbours, sections, f16, far):
    rng = np.random.default_rng(tokens * head_dim + rotary)
    dt = np.float16 if f16 else np.float32
    # rows of one projection's output, strided; norms of different sizes
    rows = (rng.standard_normal((tokens, heads + kv_heads + 1, head_dim)) * np.exp(rng.standard_normal((tokens, 1, 1)))).astype(dt)
    x = _dev(rows)
    q, k = x[:, :heads], x[:, heads:heads + kv_heads]
    wq, wk = ((1 + 0.2 * rng.standard_normal(head_dim)).astype(dt) for _ in range(2))
    pos = (far + rng.integers(0, 199, (len(sections), tokens)) * (1 if far else rng.choice([1, -1], (1, tokens)))).astype(np.int32)
    plan = mld.QkNormRope(heads, kv_heads, head_dim, rotary, mld.ROPE_NEIGHBOURS if neighbours else mld.ROPE_HALVES, sections,
                          max_timescale=1e5, rms_eps=1e-5, f16=f16)
    tt = torch.float16 if f16 else torch.float32
    qo = torch.full((tokens, heads, head_dim), float("nan"), dtype=tt, device="cuda")
    ko = torch.full((tokens, kv_heads, head_dim), float("nan"), dtype=tt, device="cuda")
    plan.run(q, k, _dev(pos), qo, ko, q_weight=_dev(wq), k_weight=_dev(wk))
    for got, src, w in ((qo, rows[:, :heads], wq), (ko, rows[:, heads:heads + kv_heads], wk)):
        want = ref.norm_rope(src, w, 1e-5, pos, rotary, neighbours, sections, 1.0, 1e5)
        # timescales are held as 32-bit floats and raised in 64 bits, angles in 2^-64 turns read to 2^-31: 2^-28 of the pair
        size = np.abs(want).max(-1, keepdims=True)
        tol = 16 * 2.0 ** -24 * size + (2.0 ** -11 * np.abs(want) + 2.0 ** -25 if f16 else 0)
        assert (np.abs(got.cpu().numpy().astype(np.float64) - want) <= tol).all()


def test_in_place_without_weights_and_without_keys(mld):
    rng = np.random.default_rng(5)
    rows = rng.standard_normal((6, 4, 64)).astype(np.float32)
    x, pos = _dev(rows), np.arange(6, dtype=np.int32)
    mld.QkNormRope(4, 0, 64, f16=False).run(x, None, _dev(pos), x)
    want = ref.norm_rope(rows, None, 0, pos[None], 64, False, [32], 1.0, 1e6)
    assert np.abs(x.cpu().numpy() - want).max() <= 16 * 2.0 ** -24 * np.abs(want).max()


@pytest.mark.parametrize("head_dim,f16", [(64, True), (128, True), (256, True), (128, False)])
def test_keys_and_values_written_in_the_same_pass_are_those_written_after_it(mld, head_dim, f16):
    rng = np.random.default_rng(head_dim)
    n, h, hk = 41, 6, 2
    dt, tt = (np.float16, torch.float16) if f16 else (np.float32, torch.float32)
    x = _dev(rng.standard_normal((n, h + 2 * hk, head_dim)).astype(dt))
    q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    w = _dev((1 + 0.1 * rng.standard_normal(head_dim)).astype(dt))
    pos, slots = _dev(np.arange(n, dtype=np.int32) + 1000), _dev(_slots(rng, n, 16, 5))
    plan = mld.QkNormRope(h, hk, head_dim, f16=f16)
    qo, qo2 = (torch.empty(n, h, head_dim, dtype=tt, device="cuda") for _ in range(2))
    ko = torch.empty(n, hk, head_dim, dtype=tt, device="cuda")
    caches = [mld.Kv4Cache(hk, head_dim, 16, 5) for _ in range(3)]
    plan.run(q, k, pos, qo, ko, q_weight=w, k_weight=w, v=v, cache=caches[0], slots=slots)
    plan.run(q, k, pos, qo2, None, q_weight=w, k_weight=w, v=v, cache=caches[1], slots=slots)
    caches[2].write(ko, v, slots)
    assert torch.equal(qo, qo2)
    assert torch.equal(caches[0].pool, caches[1].pool) and torch.equal(caches[0].pool, caches[2].pool)
    assert int(caches[0].pool.count_nonzero()) > 0


# --------------------------------------------------------------------------------------------------------- attention
def _attention_case(mld, seed, head_dim, kv_heads, group, page, lens, news, window=0, scale=0.0, spread=1.5, v_size=1.0, wide=0):
    """Runs a batch and compares every row with the restatement on what the cache holds."""
    rng = np.random.default_rng(seed)
    heads, batch = kv_heads * group, len(lens)
    per = [-(-n // page) for n in lens]
    pages = sum(per) + 3
    order = rng.permutation(pages)
    table = np.full((batch, max(max(per), wide, 1) + 1), -7, np.int32)  # entries that nobody may read
    cache = mld.Kv4Cache(kv_heads, head_dim, page, pages)
    cache.pool.fill_(0x7E)                                        # NaN scales wherever nothing is written
    kept, at = [], 0
    for b, n in enumerate(lens):
        table[b, :per[b]] = order[at:at + per[b]]
        at += per[b]
        if n == 0:
            kept.append((np.zeros((0, kv_heads, head_dim)),) * 2)
            continue
        slots = _dev((table[b][np.arange(n) // page] * page + np.arange(n) % page).astype(np.int32))
        k = rng.standard_normal((n, kv_heads, head_dim)).astype(np.float16)
        v = ((rng.standard_normal((n, kv_heads, head_dim)) + 0.3) * v_size).astype(np.float16)
        cache.write(_dev(k), _dev(v), slots)
        gk, gv = (torch.empty(n, kv_heads, head_dim, dtype=torch.float16, device="cuda") for _ in range(2))
        cache.read(slots, gk, gv)
        kept.append((gk.cpu().numpy(), gv.cpu().numpy()))
    starts = np.concatenate(([0], np.cumsum(news))).astype(np.int32)
    total = int(starts[-1])
    # rows of a wider tensor
    qw = (rng.standard_normal((total, heads + 1, head_dim)) * spread).astype(np.float16)
    q = _dev(qw)[:, 1:]
    out = torch.full((total, heads + 2, head_dim), float("nan"), dtype=torch.float16, device="cuda")
    sc = scale if scale else head_dim ** -0.5
    wants = [ref.attention(qw[starts[b]:starts[b + 1], 1:], *kept[b], news[b], sc, window) for b in range(batch)]
    one = all(m == 1 for m in news)
    args = dict() if one else dict(q_starts=_dev(starts), max_queries=max(news))
    for path in (mld.KV4_PATH_AUTO, mld.KV4_PATH_FEW_ROWS, mld.KV4_PATH_MANY_ROWS):
        out.fill_(float("nan"))
        plan = mld.Kv4Attention(cache, heads, batch + 1, table.shape[1], window=window, scale=scale, force_path=path)
        plan.run(q, _dev(table), _dev(np.int32(lens)), out[:, :heads], **args)
        first = out.clone()
        plan.run(q, _dev(table), _dev(np.int32(lens)), out[:, :heads], **args)
        assert plan.device_status() == 0
        got = out[:, :heads].cpu().numpy().astype(np.float64)
        assert np.array_equal(first[:, :heads].cpu().numpy().astype(np.float64), got), "two runs differ"
        assert bool(torch.isnan(out[:, heads:]).all()), "wrote beside the output"
        for b, (want, size) in enumerate(wants):
            r0, r1 = int(starts[b]), int(starts[b + 1])
            tol = 1.1 * 2.0 ** -11 * (np.abs(want) + size) + 2.0 ** -25
            bad = np.abs(got[r0:r1] - want) > tol
            assert not bad.any(), (path, b, lens[b], int(bad.sum()), float((np.abs(got[r0:r1] - want) / (tol + 1e-30)).max()))


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 300, 1000])
def test_one_token_over_lengths_at_the_edges_of_tiles_pages_and_chunks(mld, head_dim, n):
    _attention_case(mld, n, head_dim, 2, 4, 48, [n], [1])


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 2, 3, 5, 8, 12, 16])
def test_shared_heads(mld, head_dim, group):
    _attention_case(mld, group, head_dim, 3, group, 16, [77, 210], [1, 1])


@pytest.mark.parametrize("head_dim,kv_heads,page", [(128, 8, 64), (64, 1, 16), (256, 2, 32), (128, 1, 128)])
def test_one_long_sequence_shared_by_many_blocks(mld, head_dim, kv_heads, page):
    _attention_case(mld, 9, head_dim, kv_heads, 4, page, [20011], [1])


@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_ragged_batch_with_empty_sequences(mld, head_dim):
    lens = [0, 1, 500, 0, 16, 333, 2, 64, 1200, 7, 0]
    _attention_case(mld, 11, head_dim, 2, 4, 16, lens, [1] * len(lens))


def test_a_batch_of_nothing_but_empty_sequences(mld):
    _attention_case(mld, 12, 128, 2, 4, 16, [0, 0, 0], [1, 1, 1])


def test_many_short_sequences(mld):
    rng = np.random.default_rng(1)
    lens = [int(n) for n in rng.integers(0, 70, 300)]
    _attention_case(mld, 13, 64, 2, 2, 16, lens, [1] * 300)


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 5, 16, 100])
def test_window(mld, head_dim, window):
    _attention_case(mld, window, head_dim, 2, 3, 32, [1, 40, 333, 100, 101], [1] * 5, window=window)
    _attention_case(mld, window, head_dim, 1, 3, 16, [3, 40, 333], [3, 7, 5], window=window)


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 4, 5])
@pytest.mark.parametrize("news", [[2, 1, 2], [5, 0, 3], [17, 4, 40], [130, 1, 257]])
def test_several_new_tokens(mld, head_dim, group, news):
    # the second sequence's queries outnumber its tokens: the first of them see nothing
    lens = [max(news[0], 50), max(0, news[1] - 2), news[2] + 300]
    _attention_case(mld, sum(news), head_dim, 2, group, 32, lens, news)


@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_a_whole_prompt(mld, head_dim):
    _attention_case(mld, 21, head_dim, 2, 2, 64, [513], [513])
    _attention_case(mld, 22, head_dim, 1, 3, 16, [200, 129], [200, 128], window=70)


@pytest.mark.parametrize("head_dim,group,lens,news,window", [(128, 4, [1500, 300], [700, 65], 0), (64, 8, [700], [333], 129),
                                                             (256, 2, [1100], [600], 0), (128, 1, [900], [900], 300)])
def test_prompts_of_many_blocks(mld, head_dim, group, lens, news, window):
    _attention_case(mld, 23, head_dim, 2, group, 64, lens, news, window=window)


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 37])
def test_nan_and_infinities_at_places_that_a_row_does_not_see_stay_out_of_it(mld, head_dim, window):
    rng = np.random.default_rng(head_dim)
    n, m, hk = 300, 90, 2
    cache = mld.Kv4Cache(hk, head_dim, 32, 10)
    k, v = (rng.standard_normal((n, hk, head_dim)).astype(np.float16) for _ in range(2))
    v[250, 1, 33], v[231, 0, 0], k[280, 0, 5] = np.nan, -np.inf, np.inf
    if window:
        v[20, 0, 40] = np.nan  # seen by nobody
    cache.write(_dev(k), _dev(v), torch.arange(n, dtype=torch.int32, device="cuda"))
    q = rng.standard_normal((m, hk, head_dim)).astype(np.float16)
    at = np.arange(n - m, n)
    sees = lambda t: (at >= t) & ((at - t < window) if window else True)  # noqa: E731
    nan = np.zeros((m, hk, head_dim), bool)
    nan[sees(250), 1, 32:64] = True
    nan[sees(231), 0, :32] = True
    nan[sees(280), 0] = True
    kr, vr = np.nan_to_num(ref.quantise(k)), np.nan_to_num(ref.quantise(v))
    want, size = ref.attention(q, kr, vr, m, head_dim ** -0.5, window)
    table = torch.arange(10, dtype=torch.int32, device="cuda")[None].contiguous()
    starts = _dev(np.int32([0, m]))
    for path in (mld.KV4_PATH_FEW_ROWS, mld.KV4_PATH_MANY_ROWS):
        out = torch.zeros(m, hk, head_dim, dtype=torch.float16, device="cuda")
        mld.Kv4Attention(cache, hk, 1, 10, window=window, force_path=path).run(_dev(q), table, _dev(np.int32([n])), out, q_starts=starts,
                                                                               max_queries=m)
        got = out.cpu().numpy().astype(np.float64)
        assert np.array_equal(np.isnan(got), nan), (path, np.isnan(got).sum(), nan.sum())
        tol = 1.1 * 2.0 ** -11 * (np.abs(want) + size) + 2.0 ** -25
        assert (np.abs(got - want)[~nan] <= tol[~nan]).all()


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("lens,news,group,window", [([9000], [1], 1, 0), ([4097], [70], 4, 0), ([20011, 0, 333, 6000], [33, 4, 65, 1], 4, 0),
                                                    ([9001, 5000], [50, 130], 3, 4500), ([70], [9], 2, 0)])
def test_long_sequences_are_cut_and_joined(mld, head_dim, lens, news, group, window):
    _attention_case(mld, 41, head_dim, 2, group, 48, lens, news, window=window, wide=100)


@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_a_captured_call_cuts_anew_for_new_lengths(mld, head_dim):
    page, pages, m = 64, 160, 100
    cache = mld.Kv4Cache(1, head_dim, page, pages)
    k, v = (torch.randn(pages * page, 1, head_dim, device="cuda").half() for _ in range(2))
    cache.write(k, v, torch.arange(pages * page, dtype=torch.int32, device="cuda"))
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].contiguous()
    q = torch.randn(m, 4, head_dim, device="cuda").half()
    starts, lens, out = _dev(np.int32([0, m])), _dev(np.int32([9000])), torch.zeros_like(q)
    plan = mld.Kv4Attention(cache, 4, 1, pages, force_path=mld.KV4_PATH_MANY_ROWS)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run(q, table, lens, out, q_starts=starts, max_queries=m)
        plan.run(q, table, lens, out, q_starts=starts, max_queries=m)
    for n in (9000, 150, 10240, 100):
        lens.fill_(n)
        out.fill_(float("nan"))
        graph.replay()
        want = torch.zeros_like(q)
        torch.cuda.synchronize()
        plan.run(q, table, lens, want, q_starts=starts, max_queries=m)
        torch.cuda.synchronize()
        assert torch.equal(out, want), n
    assert plan.device_status() == 0


def test_more_heads_than_places_for_cut_blocks(mld):
    _attention_case(mld, 42, 64, 800, 1, 16, [40, 17], [3, 2], wide=260)


@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_what_is_not_finite_stays_in_its_groups_when_a_sequence_is_cut(mld, head_dim):
    rng = np.random.default_rng(head_dim)
    n, m, page = 12000, 90, 64
    pages = -(-n // page)
    cache = mld.Kv4Cache(1, head_dim, page, pages)
    k, v = (rng.standard_normal((n, 1, head_dim)).astype(np.float16) for _ in range(2))
    v[11950, 0, 33] = np.nan  # seen by the last 50 rows
    cache.write(_dev(k), _dev(v), torch.arange(n, dtype=torch.int32, device="cuda"))
    q = rng.standard_normal((m, 1, head_dim)).astype(np.float16)
    nan = np.zeros((m, 1, head_dim), bool)
    nan[np.arange(n - m, n) >= 11950, 0, 32:64] = True
    want, size = ref.attention(q, ref.quantise(k), np.nan_to_num(ref.quantise(v)), m, head_dim ** -0.5, 0)
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].contiguous()
    for path in (mld.KV4_PATH_FEW_ROWS, mld.KV4_PATH_MANY_ROWS):
        out = torch.zeros(m, 1, head_dim, dtype=torch.float16, device="cuda")
        plan = mld.Kv4Attention(cache, 1, 1, pages, force_path=path)
        plan.run(_dev(q), table, _dev(np.int32([n])), out, q_starts=_dev(np.int32([0, m])), max_queries=m)
        got = out.cpu().numpy().astype(np.float64)
        assert np.array_equal(np.isnan(got), nan), path
        assert (np.abs(got - want)[~nan] <= (1.1 * 2.0 ** -11 * (np.abs(want) + size) + 2.0 ** -25)[~nan]).all()


@pytest.mark.parametrize("head_dim,kv_heads,page", [(64, 2, 64), (128, 2, 16), (256, 1, 64)])
def test_a_hundred_runs_give_the_same_bits(mld, head_dim, kv_heads, page):
    n, m, g = 5000, 70, 4  # long enough to be cut
    cache = mld.Kv4Cache(kv_heads, head_dim, page, -(-n // page))
    k, v = (torch.randn(n, kv_heads, head_dim, device="cuda").half() for _ in range(2))
    cache.write(k, v, torch.arange(n, dtype=torch.int32, device="cuda"))
    q = (torch.randn(m, kv_heads * g, head_dim, device="cuda") * 1.5).half()
    table = torch.arange(-(-n // page), dtype=torch.int32, device="cuda")[None].contiguous()
    for path in (mld.KV4_PATH_FEW_ROWS, mld.KV4_PATH_MANY_ROWS):
        plan = mld.Kv4Attention(cache, kv_heads * g, 1, table.shape[1], force_path=path)
        outs = [torch.full_like(q, float("nan")) for _ in range(100)]
        for out in outs:
            plan.run(q, table, _dev(np.int32([n])), out, q_starts=_dev(np.int32([0, m])), max_queries=m)
        assert all(torch.equal(o, outs[0]) for o in outs) and bool(torch.isfinite(outs[0]).all())


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("news", [[1, 1], [40, 3]])
def test_sharp_and_flat_scores_and_values_of_any_size(mld, head_dim, news):
    for spread, v_size, scale in ((30.0, 1.0, 0.0), (1e-3, 1.0, 0.0), (1.5, 5000.0, 0.0), (1.5, 1e-3, 0.0), (1.5, 1.0, 0.9)):
        _attention_case(mld, 31, head_dim, 2, 4, 16, [400, 90], news, spread=spread, v_size=v_size, scale=scale)


def test_nan_in_the_cache_reaches_the_rows_that_see_it_and_no_other(mld):
    cache = mld.Kv4Cache(1, 64, 16, 4)
    k = torch.randn(64, 1, 64, device="cuda").half()
    v = k.clone()
    v[40] = float("nan")
    cache.write(k, v, torch.arange(64, dtype=torch.int32, device="cuda"))
    plan = mld.Kv4Attention(cache, 2, 3, 4)
    q = torch.randn(3, 2, 64, device="cuda").half()
    table = torch.arange(4, dtype=torch.int32, device="cuda").repeat(3, 1).contiguous()
    out = torch.zeros(3, 2, 64, dtype=torch.float16, device="cuda")
    plan.run(q, table, _dev(np.int32([40, 41, 64])), out)
    assert bool(torch.isfinite(out[0]).all()) and bool(torch.isnan(out[1:]).all())


def test_attention_on_another_stream_and_in_a_graph(mld):
    rng = np.random.default_rng(2)
    cache = mld.Kv4Cache(4, 128, 64, 40)
    n = 2500
    k, v = (_dev(rng.standard_normal((n, 4, 128)).astype(np.float16)) for _ in range(2))
    cache.write(k, v, torch.arange(n, dtype=torch.int32, device="cuda"))
    table = torch.arange(40, dtype=torch.int32, device="cuda")[None].contiguous()
    lens = _dev(np.int32([n]))
    q = _dev(rng.standard_normal((1, 16, 128)).astype(np.float16))
    want, out = torch.empty_like(q), torch.empty_like(q)
    plan = mld.Kv4Attention(cache, 16, 1, 40)
    plan.run(q, table, lens, want)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        plan.run(q, table, lens, out)
    s.synchronize()
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan.run(q, table, lens, out)
        lens.sub_(1)
    for _ in range(3):
        out.zero_()
        lens.fill_(n)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_what_does_not_fit_on_the_device_is_reported(mld):
    cache = mld.Kv4Cache(1, 64, 16, 4)
    k = torch.randn(64, 1, 64, device="cuda").half()
    cache.write(k, k, torch.arange(64, dtype=torch.int32, device="cuda"))
    plan = mld.Kv4Attention(cache, 1, 2, 2)
    q = torch.randn(2, 1, 64, device="cuda").half()
    out = torch.empty_like(q)
    good = _dev(np.int32([[0, 1], [2, 3]]))
    plan.run(q, good, _dev(np.int32([32, 20])), out)
    assert plan.device_status() == 0
    plan.run(q, _dev(np.int32([[0, 4], [2, -1]])), _dev(np.int32([32, 20])), out)
    assert plan.device_status() != 0
    assert "page" in mld.lib().mld_last_error().decode()
    plan.run(q, good, _dev(np.int32([33, -1])), out)
    assert plan.device_status() != 0
    assert "longer" in mld.lib().mld_last_error().decode()
    plan.run(q, good, _dev(np.int32([32, 20])), out, q_starts=_dev(np.int32([0, 1, 9])), max_queries=1)
    assert plan.device_status() != 0
    plan.run(q, good, _dev(np.int32([32, 20])), out)
    assert plan.device_status() == 0


# ------------------------------------------------------------------------------------------------------------- pages
@pytest.mark.parametrize("layers,pages,kv_heads,head_dim,page,count", [(1, 4, 1, 64, 16, 1), (3, 50, 3, 128, 48, 20), (2, 1300, 1, 64, 16, 600),
                                                                        (1, 9, 8, 256, 64, 4)])
def test_copies_of_pages(mld, layers, pages, kv_heads, head_dim, page, count):
    rng = np.random.default_rng(pages)
    cache = mld.Kv4Cache(kv_heads, head_dim, page, pages, layers=layers)
    cache.pool.copy_(_dev(rng.integers(0, 256, tuple(cache.pool.shape), dtype=np.uint8)))
    want = cache.pool.clone()
    order = rng.permutation(pages)
    src, dst = order[:count].copy(), order[count:2 * count]
    src[-1] = src[0]  # one page to two places
    want[:, _dev(dst)] = want[:, _dev(src)]
    cache.copy_pages(src.tolist(), dst.tolist())
    assert torch.equal(cache.pool, want)


def test_forked_sequences_part_and_compacting_keeps_them(mld):
    rng = np.random.default_rng(8)
    hk, d, page, pages = 2, 128, 16, 24
    cache = mld.Kv4Cache(hk, d, page, pages, layers=2)
    pager = mld.Kv4Pager(pages, page, 4)
    plan = mld.Kv4Attention(cache, 4, 1, pages)
    held = {}

    def append(s, n):
        slots, copies = pager.append(s, n)
        cache.copy_pages([a for a, _ in copies], [b for _, b in copies])
        k, v = (rng.standard_normal((n, hk, d)).astype(np.float16) for _ in range(2))
        for layer in range(2):
            cache.write(_dev(k), _dev(v), _dev(np.int32(slots)), layer=layer)
        held[s] = [np.concatenate((old, new)) for old, new in zip(held.get(s, (k[:0], v[:0])), (ref.quantise(k), ref.quantise(v)))]

    def check(s):
        n = pager.length(s)
        table = np.zeros((1, pages), np.int32)
        table[0, :len(pager.table(s))] = pager.table(s)
        q = rng.standard_normal((1, 4, d)).astype(np.float16)
        out = torch.empty(1, 4, d, dtype=torch.float16, device="cuda")
        plan.run(_dev(q), _dev(table), _dev(np.int32([n])), out, layer=1)
        want, size = ref.attention(q, *held[s], 1, d ** -0.5, 0)
        assert (np.abs(out.cpu().numpy() - want) <= 1.1 * 2.0 ** -11 * (np.abs(want) + size) + 2.0 ** -25).all()

    a, other = pager.open(), pager.open()
    append(other, 70)
    append(a, 53)
    b = pager.fork(a)
    held[b] = [x.copy() for x in held[a]]
    append(b, 3)
    append(a, 20)
    for s in (a, b, other):
        check(s)
    pager.truncate(a, 50)
    held[a] = [x[:50] for x in held[a]]
    append(a, 9)
    pager.close_sequence(other)
    src, dst = pager.compact()
    assert src
    cache.copy_pages(src, dst)
    for s in (a, b):
        check(s)


# ---------------------------------------------------------------------------------------------------------- refusals
def test_refusals_with_tensors(mld):
    cache = mld.Kv4Cache(2, 64, 16, 4)
    q = torch.zeros(1, 4, 64, dtype=torch.float16, device="cuda")
    plan = mld.Kv4Attention(cache, 4, 1, 4)
    table, lens = torch.zeros(1, 4, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    for bad in (dict(q=q.float()), dict(q=q[:, :2]), dict(page_table=table[:, :2].contiguous()), dict(lens=lens.long()),
                dict(q_starts=lens)):
        args = {"q": q, "page_table": table, "lens": lens, "out": torch.empty_like(q), **bad}
        with pytest.raises(ValueError):
            plan.run(**args)
    with pytest.raises(mld.MldError) as e:
        plan.run(q, table, lens, torch.empty_like(q), max_queries=2)
    assert e.value.status == mld.INVALID_ARGUMENT
    with pytest.raises(ValueError):
        mld.Kv4Cache(2, 64, 16, 4, pool=torch.zeros(5, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError):
        mld.QkNormRope(4, 2, 64).run(q, q, torch.zeros(1, dtype=torch.int32, device="cuda"), q)
    k = torch.zeros(1, 2, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(mld.MldError):  # neither a key output nor a cache
        mld.QkNormRope(4, 2, 64).run(q, k, torch.zeros(1, dtype=torch.int32, device="cuda"), q)
    with pytest.raises(mld.MldError):  # a plan of another shape
        mld.QkNormRope(4, 2, 128).desc and mld.QkNormRope(2, 1, 64).run(
            q[:, :2], k[:, :1], torch.zeros(1, dtype=torch.int32, device="cuda"), q[:, :2], v=k[:, :1], cache=cache, slots=lens)
    for src, dst in (([0], [4]), ([-1], [0]), ([0, 1], [1, 2]), ([0, 1], [2, 2]), ([1], [1])):
        with pytest.raises(mld.MldError) as e:
            cache.copy_pages(src, dst)
        assert e.value.status == mld.INVALID_ARGUMENT
    io = mld.binding.Kv4AttnIo(q.data_ptr() + 2, 256, cache.address(), table.data_ptr(), lens.data_ptr(), None, 1, 1, 1, q.data_ptr(), 256)
    assert mld.lib().mld_kv4_attn_run(plan._h, ctypes.byref(io), None) == mld.INVALID_ARGUMENT
