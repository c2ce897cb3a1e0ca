"""The operators around the 4-bit cache run together as a server runs them (examples/paged_serving.py)."""
import importlib.util
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from tests import kv4_ref as ref

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PATH = os.path.join(ROOT, "examples", "paged_serving.py")


@pytest.fixture(scope="module")
def serving():
    spec = importlib.util.spec_from_file_location("paged_serving", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _tokens(n, seed, d_model=1024):
    return torch.randn(n, d_model, generator=torch.Generator().manual_seed(seed)).half().cuda()


def test_a_forked_sequence_goes_on_as_its_origin_would_have(serving):
    a, b = serving.Server(), serving.Server()
    x, more, other = _tokens(77, 1), _tokens(5, 2), _tokens(5, 3)
    s, t = a.pager.open(), b.pager.open()
    a.prompt(s, x)
    b.prompt(t, x)
    fork = a.pager.fork(s)
    for i in range(5):  # both branches at once in one server, the one with `more` alone in the other
        branch = a.step([(s, other[i:i + 1]), (fork, more[i:i + 1])])[1]
        alone = b.step([(t, more[i:i + 1])])[0]
        torch.testing.assert_close(branch, alone, rtol=2 ** -6, atol=2 ** -6)
    a.check()
    b.check()


def test_closing_and_compacting_change_no_answer(serving):
    def run(compact):
        server = serving.Server(pages=24)
        ss = [server.pager.open() for _ in range(3)]
        for i, s in enumerate(ss):
            server.prompt(s, _tokens(150 + 31 * i, i))
        server.pager.close_sequence(ss[0])
        moved = server.compact() if compact else 0
        out = server.step([(ss[1], _tokens(1, 9)), (ss[2], _tokens(3, 10))])
        server.check()
        return moved, out
    (moved, one), (_, two) = run(True), run(False)
    assert moved > 0
    assert all(torch.equal(x, y) for x, y in zip(one, two))


@pytest.mark.parametrize("most", [512, 64])
def test_a_prompt_against_the_formulas(serving, most):
    """One layer, from its projections on: norm, rotation, rounding to 4 bits, attention, all in 64 bits."""
    server = serving.Server(layers=1, most=most)
    layer, n = server.layers[0], 150
    x, seen = _tokens(n, 4), []
    inner = layer["qkv"]
    layer["qkv"] = lambda y: seen.append(inner(y)) or seen[-1]
    outer, heads_out = layer["out"], []
    layer["out"] = lambda o: heads_out.append(o.clone()) or outer(o)
    server.prompt(server.pager.open(), x)
    server.check()
    h, hk, d = server.heads, server.kv_heads, server.head_dim
    qkv = torch.cat(seen).view(n, h + 2 * hk, d).cpu().numpy()
    weights = [layer[w].cpu().numpy() for w in ("q_norm", "k_norm")]
    at = np.arange(n)[None]
    q, k = (ref.norm_rope(p, w, 1e-6, at, d, False, [d // 2], 1.0, 1e6)
            for p, w in zip((qkv[:, :h], qkv[:, h:h + hk]), weights))
    # Queries are rounded to fp16 (2^-11 of a score's terms); keys may fall on the other side of a code's boundary by the
    # rounding of 32-bit arithmetic: what the cache holds is read back.
    pages = server.pager.table(0)
    slots = torch.tensor([pages[i // 32] * 32 + i % 32 for i in range(n)], dtype=torch.int32, device="cuda")
    keys, values = (torch.empty(n, hk, d, dtype=torch.float16, device="cuda") for _ in range(2))
    server.cache.read(slots, keys, values)
    keys, values = keys.cpu().numpy().astype(np.float64), values.cpu().numpy().astype(np.float64)
    assert np.array_equal(values, ref.quantise(qkv[:, h + hk:]))
    assert (keys != ref.quantise(k)).mean() < 1e-2
    q = q.astype(np.float16).astype(np.float64)
    want, size = ref.attention(q, keys, values, n, d ** -0.5, 0)
    got = torch.cat(heads_out).view(n, h, d).cpu().numpy().astype(np.float64)
    # A query's rounding may differ by one unit, 2^-10 of its largest value, from the kernel's: the score moves by at most
    # 2^-10 |q| |k| / sqrt(d), which moves a mean of v by twice that of sum(p |v|); beside it the roundings of the weights and of
    # the output, 2^-11 each, a tenth on top.
    score = 2.0 ** -10 * np.linalg.norm(q, axis=-1).max() * np.linalg.norm(keys, axis=-1).max() * d ** -0.5
    assert (np.abs(got - want) <= (2.2 * score + 1.1 * 2 ** -11) * size + 1.1 * 2 ** -11 * np.abs(want) + 1e-7).all()


def test_the_example_runs():
    out = subprocess.run([sys.executable, PATH, "--layers", "2", "--d-model", "1024", "--prompt", "600", "--steps", "6"],
                         capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert out.returncode == 0, out.stderr[-2000:]
    assert "ms a step" in out.stdout and "pages moved" in out.stdout
