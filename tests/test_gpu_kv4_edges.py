"""Edges of the 4-bit cache's operators: values that are not finite, sizes near 2^31, batches of very uneven sequences.

Tolerances are those of the operators' other tests: attention 2^-11 of the output and of sum(p |v|), a tenth on top; rotation a
handful of roundings of 2^-24 of a row's size and of the output's type."""
import ctypes

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


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("head_dim,rotary", [(64, 16), (128, 64), (256, 240), (64, 0), (128, 128)])
def test_what_is_not_finite_in_a_head_changes_only_what_the_formula_says(mld, head_dim, rotary, neighbours, weighted, f16):
    rng = np.random.default_rng(head_dim + rotary)
    dt, tt = (np.float16, torch.float16) if f16 else (np.float32, torch.float32)
    n, h = 12, 3
    x = rng.standard_normal((n, h, head_dim)).astype(dt)
    places = [0, 1, rotary // 2, max(rotary - 1, 0), rotary % head_dim, (rotary + 1) % head_dim, (rotary + 6) % head_dim, head_dim - 1]
    for i, (at, value) in enumerate(zip(places + places[:2], [np.inf, -np.inf, np.nan] * 4)):
        x[i, 1, at] = value
    pos = rng.integers(1, 1000, (1, n)).astype(np.int32)
    w = (1 + 0.1 * rng.standard_normal(head_dim)).astype(dt) if weighted else None
    plan = mld.QkNormRope(h, h, head_dim, rotary, mld.ROPE_NEIGHBOURS if neighbours else mld.ROPE_HALVES, rms_eps=1e-5, f16=f16)
    qo, ko = (torch.zeros(n, h, head_dim, dtype=tt, device="cuda") for _ in range(2))
    wd = None if w is None else _dev(w)
    plan.run(_dev(x), _dev(x), _dev(pos[0]), qo, ko, q_weight=wd, k_weight=wd)
    with np.errstate(invalid="ignore"):
        want = ref.norm_rope(x, w, 1e-5, pos, rotary, neighbours, [rotary // 2], 1.0, 1e6)
    size = np.where(np.isfinite(want), np.abs(want), 0).max(-1, keepdims=True)
    for got in (qo.cpu().numpy().astype(np.float64), ko.cpu().numpy().astype(np.float64)):
        finite = np.isfinite(want)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
        tol = 16 * 2.0 ** -24 * size + (2.0 ** -11 * np.abs(want) + 2.0 ** -25 if f16 else 0 * want)
        assert (np.abs(got[finite] - want[finite]) <= tol[finite]).all()


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


def test_a_sequence_of_almost_2_31_tokens(mld):
    """One page of keys and values 2^26 times over, then another one as often."""
    rng = np.random.default_rng(7)
    d, page, entries = 64, 16, (1 << 27) - 1
    cache = mld.Kv4Cache(1, d, page, 2)
    k, v = (rng.standard_normal((2 * page, 1, d)).astype(np.float16) for _ in range(2))
    v[page:] += np.float16(2)
    cache.write(_dev(k), _dev(v), torch.arange(2 * page, dtype=torch.int32, device="cuda"))
    table = torch.zeros(1, entries, dtype=torch.int32, device="cuda")
    table[:, entries // 2:] = 1
    q = rng.standard_normal((1, 1, d)).astype(np.float16)
    out = torch.zeros(1, 1, d, dtype=torch.float16, device="cuda")
    plan = mld.Kv4Attention(cache, 1, 1, entries, force_path=mld.KV4_PATH_FEW_ROWS)
    plan.run(_dev(q), table, _dev(np.int32([entries * page])), out)
    assert plan.device_status() == 0
    want, size = ref.attention(q, ref.quantise(k), ref.quantise(v), 1, d ** -0.5, 0)
    # A warp adds 2^27 / (148 * 12) products of 16 tokens up in 32 bits: 2^-23 of the sum each, if all err to one side.
    tol = 2 ** 27 / (148 * 12) * 2.0 ** -23 * size + 2.0 ** -10
    assert (np.abs(out.cpu().numpy() - want) <= tol).all()


def _time(call):
    """Microseconds of a call, the smallest of five means of ten."""
    for _ in range(3):
        call()
    best = float("inf")
    for _ in range(5):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        for _ in range(10):
            call()
        end.record()
        end.synchronize()
        best = min(best, begin.elapsed_time(end) * 100)
    return best


def _timed_batch(mld, kv_heads, lens, news, pages=0):
    """A batch over one pool of random codes, page tables that share its pages; the call."""
    page, d, g = 64, 128, 4
    cache = mld.Kv4Cache(kv_heads, d, page, 512)
    k = torch.randn(512 * page, kv_heads, d, device="cuda").half()
    cache.write(k, k, torch.arange(512 * page, dtype=torch.int32, device="cuda"))
    pages = max(pages, -(-max(lens) // page))
    table = torch.randint(0, 512, (len(lens), pages), dtype=torch.int32, device="cuda")
    starts = np.concatenate(([0], np.cumsum(news))).astype(np.int32)
    q = torch.randn(int(starts[-1]), kv_heads * g, d, device="cuda").half()
    plan, out = mld.Kv4Attention(cache, kv_heads * g, len(lens), pages), torch.empty_like(q)
    lens, starts, longest = _dev(np.int32(lens)), _dev(starts), max(news)
    return lambda: plan.run(q, table, lens, out, q_starts=starts, max_queries=longest)


def test_one_long_sequence_among_many_short_ones(mld):
    lens = [int(n) for n in np.random.default_rng(3).integers(1, 33, 147)]
    lens.insert(70, 108000)
    _attention_case(mld, 51, 128, 1, 4, 64, lens, [1] * 148)


@pytest.mark.parametrize("kv_heads,shorter,longest", [(1, 147, 108000), (8, 17, 13000)])
def test_a_long_sequence_takes_no_longer_for_short_ones_beside_it(mld, kv_heads, shorter, longest):
    alone = _time(_timed_batch(mld, kv_heads, [longest], [1]))
    beside = _time(_timed_batch(mld, kv_heads, [20] * (shorter // 2) + [longest] + [20] * (shorter - shorter // 2), [1] * (shorter + 1)))
    assert beside < 3 * alone + 20, (alone, beside)


@pytest.mark.parametrize("history,times", [(131072, 4), (1000, 3)])
def test_a_chunk_of_a_prompt_beside_many_single_tokens(mld, history, times):
    """The rows of a call are counted as they are, not as if every sequence had as many as the one with the most."""
    chunk = _time(_timed_batch(mld, 8, [4000], [2048]))
    tokens = _time(_timed_batch(mld, 8, [1000] * 127 + [history], [1] * 128))
    both = _time(_timed_batch(mld, 8, [1000] * 127 + [history, 4000], [1] * 128 + [2048]))
    assert both < times * (chunk + tokens), (chunk, tokens, both)


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 60, 1 << 20])
def test_a_window_wider_than_any_sequence_hides_nothing(mld, head_dim, window):
    # the queries outnumber the tokens of the first sequence: the first of them see nothing
    _attention_case(mld, 61, head_dim, 2, 4, 32, [3, 300, 0], [70, 5, 2], window=window)
    _attention_case(mld, 62, head_dim, 1, 2, 16, [100, 5000], [120, 40], window=window, wide=400)


def test_one_row_for_all_tokens_may_be_read_and_not_written(mld):
    rng = np.random.default_rng(1)
    n, h, hk, d = 9, 4, 2, 64
    row = rng.standard_normal((1, h + 2 * hk, d)).astype(np.float16)
    x = _dev(row).expand(n, -1, -1)
    pos, slots = torch.arange(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")
    plan, outs = mld.QkNormRope(h, hk, d), []
    for rows in (x, x.contiguous()):
        cache = mld.Kv4Cache(hk, d, 16, 1)
        q, k = torch.zeros(n, h, d, dtype=torch.float16, device="cuda"), torch.zeros(n, hk, d, dtype=torch.float16, device="cuda")
        plan.run(rows[:, :h], rows[:, h:h + hk], pos, q, k, v=rows[:, h + hk:], cache=cache, slots=slots)
        again = mld.Kv4Cache(hk, d, 16, 1)
        again.write(rows[:, h:h + hk], rows[:, h + hk:], slots)
        outs.append((q, k, cache.pool, again.pool))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    for q, k in ((torch.zeros(1, h, d, dtype=torch.float16, device="cuda").expand(n, -1, -1), outs[0][1]),
                 (outs[0][0], torch.zeros(1, hk, d, dtype=torch.float16, device="cuda").expand(n, -1, -1))):
        with pytest.raises(mld.MldError) as e:
            plan.run(x[:, :h], x[:, h:h + hk], pos, q, k)
        assert e.value.status == mld.INVALID_ARGUMENT


def test_any_tensor_in_host_memory_is_refused(mld):
    """What a pager answers is easily made a tensor without a device."""
    n, h, hk, d = 3, 4, 2, 64
    cache = mld.Kv4Cache(hk, d, 16, 4)
    rope, attention = mld.QkNormRope(h, hk, d), mld.Kv4Attention(cache, h, 1, 4)
    q, k = (torch.zeros(n, heads, d, dtype=torch.float16, device="cuda") for heads in (h, hk))
    ints, w = torch.arange(n, dtype=torch.int32, device="cuda"), torch.ones(d, dtype=torch.float16, device="cuda")
    calls = [(cache.write, dict(k=k, v=k, slots=ints)), (cache.read, dict(slots=ints, k=k.clone(), v=k.clone())),
             (rope.run, dict(q=q, k=k, positions=ints, q_out=q.clone(), k_out=k.clone(), q_weight=w, k_weight=w, v=k, cache=cache,
                             slots=ints)),
             (attention.run, dict(q=q, page_table=torch.zeros(1, 4, dtype=torch.int32, device="cuda"), lens=ints[:1], out=q.clone(),
                                  q_starts=_dev(np.int32([0, n])), max_queries=n))]
    for call, args in calls:
        for name, t in args.items():
            if isinstance(t, torch.Tensor):
                with pytest.raises(ValueError, match="GPU"):
                    call(**{**args, name: t.cpu()})
        call(**args)
    assert attention.device_status() == 0


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_a_plan_is_run_on_its_own_device_and_asked_from_any(mld):
    with torch.cuda.device(1):
        cache = mld.Kv4Cache(1, 64, 16, 4, device="cuda:1")
        plan = mld.Kv4Attention(cache, 1, 1, 4)
        q = torch.zeros(1, 1, 64, dtype=torch.float16, device="cuda:1")
        table, lens = torch.full((1, 4), 9, dtype=torch.int32, device="cuda:1"), torch.full((1,), 40, dtype=torch.int32, device="cuda:1")
        plan.run(q, table, lens, torch.empty_like(q), stream=torch.cuda.Stream())
    with torch.cuda.device(0):
        assert plan.device_status() != 0 and plan.device_status() == 0
        assert torch.cuda.current_device() == 0
        io = mld.binding.Kv4AttnIo(q.data_ptr(), 64, cache.address(), table.data_ptr(), lens.data_ptr(), None, 1, 1, 1, q.data_ptr(), 64)
        assert mld.lib().mld_kv4_attn_run(plan._h, ctypes.byref(io), None) == mld.INVALID_ARGUMENT


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("wide", [0, 400])
def test_batches_of_sequences_with_very_different_rows(mld, head_dim, wide):
    """Blocks of rows are found by their number: short and long sequences, some without rows, in any order; cut or not."""
    rng = np.random.default_rng(head_dim)
    news = [0, 1, 300, 1, 0, 0, 700, 2, 300, 1] + [1] * 60 + [0, 257, 256, 255, 0]
    lens = [int(n + rng.integers(0, 200)) for n in news]
    _attention_case(mld, 71, head_dim, 2, 3, 16, lens, news, wide=wide)
    order = rng.permutation(len(news))
    _attention_case(mld, 72, head_dim, 1, 1, 32, [lens[i] for i in order], [news[i] for i in order], wide=wide // 2)


def test_row_ranges_that_overlap_or_descend_are_reported_and_write_nothing_beside_the_output(mld):
    cache = mld.Kv4Cache(1, 64, 64, 80)
    k = torch.randn(80 * 64, 1, 64, device="cuda").half()
    cache.write(k, k, torch.arange(80 * 64, dtype=torch.int32, device="cuda"))
    n, batch = 600, 40
    q = torch.randn(n, 1, 64, device="cuda").half()
    good = _dev(np.linspace(0, n, batch + 1).astype(np.int32))
    for pages in (40, 80):  # whole blocks, and blocks that may be cut
        table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(batch, 1).contiguous()
        lens = torch.full((batch,), pages * 64, dtype=torch.int32, device="cuda")
        for path in (mld.KV4_PATH_FEW_ROWS, mld.KV4_PATH_MANY_ROWS):
            plan = mld.Kv4Attention(cache, 1, batch, pages, force_path=path)
            want = torch.full((n + 2, 1, 64), 7.0, dtype=torch.float16, device="cuda")
            plan.run(q, table, lens, want[1:-1], q_starts=good, max_queries=n)
            assert plan.device_status() == 0
            for bad in (np.arange(batch + 1) % 2 * n, np.where(np.arange(batch + 1) % 2, 2**31 - 1, -2**31), np.arange(batch + 1)[::-1] * 15,
                        np.arange(batch + 1) % 2 * 300):
                out = torch.full((n + 2, 1, 64), 7.0, dtype=torch.float16, device="cuda")
                plan.run(q, table, lens, out[1:-1], q_starts=_dev(bad.astype(np.int32)), max_queries=n)
                assert plan.device_status() != 0
                assert bool((out[[0, -1]] == 7).all())
            out = torch.full_like(want, 7.0)
            plan.run(q, table, lens, out[1:-1], q_starts=good, max_queries=n)
            assert plan.device_status() == 0 and torch.equal(out, want)


@pytest.mark.parametrize("head_dim,heads,kv_heads", [(128, 32, 8), (64, 6, 3), (256, 8, 1)])
def test_how_many_tokens_a_call_has_changes_no_token(mld, head_dim, heads, kv_heads):
    """Few tokens are spread over blocks by their heads, many are not."""
    n, page = 1400, 64
    x = torch.randn(n, heads + 2 * kv_heads, head_dim, device="cuda").half()
    w = (1 + 0.1 * torch.randn(head_dim, device="cuda")).half()
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    plan, outs = mld.QkNormRope(heads, kv_heads, head_dim), []
    for some in (n, 600, 290, 75, 1):
        cache = mld.Kv4Cache(kv_heads, head_dim, page, -(-n // page))
        q, k, v = (torch.zeros(n, h, head_dim, dtype=torch.float16, device="cuda") for h in (heads, kv_heads, kv_heads))
        for at in range(0, n, some):
            part = slice(at, min(n, at + some))
            y = x[part]
            plan.run(y[:, :heads], y[:, heads:heads + kv_heads], pos[part], q[part], q_weight=w, k_weight=w, v=y[:, heads + kv_heads:],
                     cache=cache, slots=pos[part])
            cache.read(pos[part], k[part], v[part])
        outs.append((q, k, v, cache.pool))
    for out in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(out, outs[0]))


@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("head_dim,rotary", [(64, 64), (128, 32), (256, 256)])
@pytest.mark.parametrize("tokens", [1, 90, 700])
def test_queries_and_keys_of_one_projection_in_place(mld, tokens, head_dim, rotary, neighbours):
    h, hk = 6, 2
    x = torch.randn(tokens, h + 2 * hk, head_dim, device="cuda").half()
    wq, wk = ((1 + 0.2 * torch.randn(head_dim, device="cuda")).half() for _ in range(2))
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda") + 77
    slots = torch.arange(tokens, dtype=torch.int32, device="cuda")
    plan = mld.QkNormRope(h, hk, head_dim, rotary, mld.ROPE_NEIGHBOURS if neighbours else mld.ROPE_HALVES)
    q, k = torch.empty(tokens, h, head_dim, dtype=torch.float16, device="cuda"), torch.empty(tokens, hk, head_dim, dtype=torch.float16, device="cuda")
    caches = [mld.Kv4Cache(hk, head_dim, 16, -(-tokens // 16)) for _ in range(2)]
    y = x.clone()
    plan.run(x[:, :h], x[:, h:h + hk], pos, q, k, q_weight=wq, k_weight=wk, v=x[:, h + hk:], cache=caches[0], slots=slots)
    plan.run(y[:, :h], y[:, h:h + hk], pos, y[:, :h], y[:, h:h + hk], q_weight=wq, k_weight=wk, v=y[:, h + hk:], cache=caches[1], slots=slots)
    assert torch.equal(y[:, :h], q) and torch.equal(y[:, h:h + hk], k) and torch.equal(y[:, h + hk:], x[:, h + hk:])
    assert torch.equal(caches[0].pool, caches[1].pool)
    want = ref.norm_rope(x[:, :h].cpu().numpy(), wq.cpu().numpy(), 1e-6, pos.cpu().numpy()[None], rotary, neighbours, [rotary // 2], 1.0, 1e6)
    tol = 16 * 2.0 ** -24 * np.abs(want).max(-1, keepdims=True) + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
    assert (np.abs(y[:, :h].cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_fp32_keys_of_neighbouring_pairs_in_the_cache(mld, head_dim):
    n, h, hk = 53, 4, 2
    rng = np.random.default_rng(head_dim)
    x = rng.standard_normal((n, h + 2 * hk, head_dim)).astype(np.float32)
    w = (1 + 0.2 * rng.standard_normal(head_dim)).astype(np.float32)
    pos = np.arange(n, dtype=np.int32) + 500
    plan = mld.QkNormRope(h, hk, head_dim, head_dim // 2, mld.ROPE_NEIGHBOURS, f16=False)
    cache, slots, xd = mld.Kv4Cache(hk, head_dim, 16, 5), torch.arange(n, dtype=torch.int32, device="cuda") + 9, _dev(x)
    q, k = torch.empty(n, h, head_dim, device="cuda"), torch.empty(n, hk, head_dim, device="cuda")
    plan.run(xd[:, :h], xd[:, h:h + hk], _dev(pos), q, k, q_weight=_dev(w), k_weight=_dev(w), v=xd[:, h + hk:], cache=cache, slots=slots)
    want = ref.norm_rope(x[:, h:h + hk], w, 1e-6, pos[None], head_dim // 2, True, [head_dim // 4], 1.0, 1e6)
    got = k.cpu().numpy()
    assert (np.abs(got - want) <= 16 * 2.0 ** -24 * np.abs(want).max(-1, keepdims=True)).all()
    gk, gv = (torch.empty(n, hk, head_dim, dtype=torch.float16, device="cuda") for _ in range(2))
    cache.read(slots, gk, gv)
    assert np.array_equal(gk.cpu().numpy().astype(np.float64), ref.quantise(got))
    assert np.array_equal(gv.cpu().numpy().astype(np.float64), ref.quantise(x[:, h + hk:]))


@pytest.mark.parametrize("head_dim,kv_heads,page", [(128, 8, 64), (64, 4, 16), (256, 2, 128)])
def test_pages_behind_the_first_gigabytes(mld, head_dim, kv_heads, page):
    """The last pages of the second layer of a cache of 10 GB against the first ones of a small one."""
    page_bytes = kv_heads * page * head_dim * 18 // 16
    pages, n, m = (5 << 30) // page_bytes, 700, 150
    large, small = mld.Kv4Cache(kv_heads, head_dim, page, pages, layers=2), mld.Kv4Cache(kv_heads, head_dim, page, 60)
    k, v = (torch.randn(n, kv_heads, head_dim, device="cuda").half() for _ in range(2))
    there = -(-n // page)
    last = pages - 1 - torch.arange(there, dtype=torch.int32, device="cuda")
    at = torch.arange(n, dtype=torch.int32, device="cuda")
    far = last[(at // page).long()] * page + at % page
    large.write(k, v, far, layer=1)
    small.write(k, v, at)
    q = torch.randn(m, kv_heads * 4, head_dim, device="cuda").half()
    table = torch.zeros(1, 60, dtype=torch.int32, device="cuda")
    outs, first = [], torch.arange(there, dtype=torch.int32, device="cuda")

    def attend(cache, layer, pages_of):
        table[0, :there] = pages_of
        for path in (mld.KV4_PATH_FEW_ROWS, mld.KV4_PATH_MANY_ROWS):
            out = torch.zeros_like(q)
            mld.Kv4Attention(cache, kv_heads * 4, 1, 60, force_path=path).run(q, table, _dev(np.int32([n])), out,
                                                                              q_starts=_dev(np.int32([0, m])), max_queries=m, layer=layer)
            outs.append(out)

    attend(small, 0, first)
    attend(large, 1, last)
    large.copy_pages(last.tolist(), (last - 100).tolist())
    attend(large, 1, last - 100)
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3]) and torch.equal(outs[0], outs[4]) and torch.equal(outs[1], outs[5])
    assert int(large.pool[0].view(torch.int64).count_nonzero()) == 0
    read = [torch.empty_like(k) for _ in range(4)]
    large.read(far, *read[:2], layer=1)
    small.read(at, *read[2:])
    assert torch.equal(read[0], read[2]) and torch.equal(read[1], read[3])
