"""The host side of the 4-bit cache: sizes, refusals that need no GPU, the pager."""
import ctypes

import numpy as np
import pytest


@pytest.fixture(scope="module")
def mld():
    import __graft_entry__ as g
    g.build()
    return g.import_package()


def test_sizes(mld):
    d = mld.binding.Kv4Desc(8, 128, 64, 10)
    assert mld.lib().mld_kv4_page_bytes(ctypes.byref(d)) == 8 * 64 * 144
    assert mld.lib().mld_kv4_pool_bytes(ctypes.byref(d)) == 10 * 8 * 64 * 144


@pytest.mark.parametrize("kv_heads,head_dim,page,pages", [(0, 128, 64, 1), (1, 96, 64, 1), (1, 128, 8, 1), (1, 128, 24, 1), (1, 128, 64, 0),
                                                          (1, 128, 64, 1 << 26), (2000, 128, 64, 1)])
def test_bad_caches_are_refused(mld, kv_heads, head_dim, page, pages):
    d = mld.binding.Kv4Desc(kv_heads, head_dim, page, pages)
    assert mld.lib().mld_kv4_pool_bytes(ctypes.byref(d)) == 0
    a = mld.binding.Kv4AttnDesc(d, max(kv_heads, 1), 1, 1, 0, 0.0, -1)
    h = ctypes.c_void_p()
    assert mld.lib().mld_kv4_attn_plan_create(ctypes.byref(a), ctypes.byref(h)) == mld.INVALID_ARGUMENT
    assert mld.lib().mld_kv4_copy_pages(ctypes.byref(d), None, 1, 0, None, None, 1, None) == mld.INVALID_ARGUMENT


@pytest.mark.parametrize("change", [dict(heads=3), dict(heads=0), dict(max_batch=0), dict(max_batch=1025), dict(max_pages=0), dict(window=-1),
                                    dict(scale=float("nan")), dict(scale=-1.0), dict(force_path=3)])
def test_bad_attention_plans_are_refused(mld, change):
    d = dict(heads=4, max_batch=1, max_pages=4, window=0, scale=0.0, force_path=0) | change
    a = mld.binding.Kv4AttnDesc(mld.binding.Kv4Desc(2, 128, 64, 10), d["heads"], d["max_batch"], d["max_pages"], d["window"], d["scale"], -1,
                                d["force_path"])
    h = ctypes.c_void_p()
    assert mld.lib().mld_kv4_attn_plan_create(ctypes.byref(a), ctypes.byref(h)) == mld.INVALID_ARGUMENT


@pytest.mark.parametrize("args", [dict(head_dim=80), dict(rotary_dim=8), dict(rotary_dim=144), dict(sections=[10]), dict(sections=[70, -6]),
                                  dict(pairing=2), dict(min_timescale=0.0), dict(max_timescale=float("inf")), dict(rms_eps=-1.0), dict(heads=-1)])
def test_bad_rotation_plans_are_refused(mld, args):
    a = dict(heads=4, kv_heads=2, head_dim=128) | args
    with pytest.raises(mld.MldError) as e:
        mld.QkNormRope(**a)
    assert e.value.status == mld.INVALID_ARGUMENT


def test_rotation_plan_needs_no_gpu_and_refuses_calls_without_tensors(mld):
    plan = mld.QkNormRope(4, 2, 128)
    io = mld.binding.QkRopeIo()
    assert mld.lib().mld_qk_rope_run(plan._h, ctypes.byref(io), 0, None) == mld.OK
    assert mld.lib().mld_qk_rope_run(plan._h, ctypes.byref(io), 1, None) == mld.INVALID_ARGUMENT
    io.q = io.q_out = io.k = io.k_out = io.positions = 4096
    io.q_stride = io.q_out_stride = 512
    io.k_stride = io.k_out_stride = 255      # shorter than a token, and not whole 16 bytes
    assert mld.lib().mld_qk_rope_run(plan._h, ctypes.byref(io), 2, None) == mld.INVALID_ARGUMENT
    io.k_stride = 256
    io.k_out_stride = 248
    assert mld.lib().mld_qk_rope_run(plan._h, ctypes.byref(io), 2, None) == mld.INVALID_ARGUMENT


class Model:
    """A pager by the book: every sequence owns a list of token names; every page a list of what was written to it."""

    def __init__(self, pages, page):
        self.page, self.content, self.seqs = page, [[None] * page for _ in range(pages)], {}

    def check(self, pager):
        held = set()
        for s, tokens in self.seqs.items():
            assert pager.length(s) == len(tokens)
            table = pager.table(s)
            assert len(table) == -(-len(tokens) // self.page) and len(set(table)) == len(table)
            held |= set(table)
            for i, name in enumerate(tokens):
                assert self.content[table[i // self.page]][i % self.page] == name
        assert pager.free_pages() == len(self.content) - len(held)


@pytest.mark.parametrize("seed", range(8))
def test_pager_against_a_model(mld, seed):
    rng = np.random.default_rng(seed)
    pages, page, most = int(rng.integers(3, 40)), int(rng.choice([16, 32])), int(rng.integers(1, 7))
    pager, model, name = mld.Kv4Pager(pages, page, most), Model(pages, page), 0

    def copy(pairs):
        old = {a: list(model.content[a]) for a, _ in pairs}
        assert not {a for a, _ in pairs} & {b for _, b in pairs} and len({b for _, b in pairs}) == len(pairs)
        for a, b in pairs:
            model.content[b] = old[a]

    for _ in range(400):
        what = rng.choice(["open", "append", "append", "append", "fork", "truncate", "close", "compact"])
        some = list(model.seqs)
        s = some[rng.integers(len(some))] if some else None
        if what in ("open", "fork") and (what == "open" or s is not None):
            if len(some) == most:
                with pytest.raises(mld.MldError) as e:
                    pager.open() if what == "open" else pager.fork(s)
                assert e.value.status == mld.OUT_OF_RANGE
            elif what == "open":
                model.seqs[pager.open()] = []
            else:
                model.seqs[pager.fork(s)] = list(model.seqs[s])
        elif what == "append" and s is not None:
            n = int(rng.integers(0, 3 * page))
            try:
                slots, pairs = pager.append(s, n)
            except mld.MldError as e:
                assert e.status == mld.OUT_OF_RANGE
            else:
                copy(pairs)
                for at in slots:
                    model.content[at // page][at % page] = name
                    model.seqs[s].append(name)
                    name += 1
        elif what == "truncate" and s is not None:
            n = int(rng.integers(0, len(model.seqs[s]) + 1))
            pager.truncate(s, n)
            del model.seqs[s][n:]
        elif what == "close" and s is not None:
            pager.close_sequence(s)
            del model.seqs[s]
        elif what == "compact":
            most_moves = int(rng.integers(0, pages + 1))
            src, dst = pager.compact(most_moves)
            assert len(src) <= most_moves and all(a > b for a, b in zip(src, dst))
            copy(list(zip(src, dst)))
            if most_moves == pages:
                held = {p for q in model.seqs for p in pager.table(q)}
                assert held == set(range(len(held)))
        model.check(pager)


def test_pager_refusals(mld):
    for args in ((0, 16, 1), (4, 8, 1), (4, 20, 1), (4, 16, 0), (1 << 27, 16, 1)):
        with pytest.raises(mld.MldError) as e:
            mld.Kv4Pager(*args)
        assert e.value.status == mld.INVALID_ARGUMENT
    p = mld.Kv4Pager(2, 16, 2)
    s = p.open()
    for call in (lambda: p.length(1), lambda: p.append(-1, 1), lambda: p.fork(5), lambda: p.truncate(s, 1), lambda: p.close_sequence(1),
                 lambda: p.append(s, -1), lambda: p.table(7)):
        with pytest.raises(mld.MldError) as e:
            call()
        assert e.value.status == mld.INVALID_ARGUMENT
    with pytest.raises(mld.MldError) as e:
        p.append(s, 33)
    assert e.value.status == mld.OUT_OF_RANGE and p.length(s) == 0 and p.free_pages() == 2
