"""Products on codes whose tensors do not fit are refused by the binding, without a GPU: nothing of them reaches the library."""
import pytest
import torch


@pytest.fixture(scope="module")
def mld():
    import __graft_entry__ as g
    g.build()
    return g.import_package()


@pytest.fixture
def call(mld, monkeypatch):
    """run_codes of a plan that holds nothing, with tensors in host memory that count as the GPU's; what the library would have got."""
    calls = []

    class Library:
        @staticmethod
        def mld_fc_run_codes(*args):
            calls.append(args)
            return mld.OK

    monkeypatch.setattr(mld.binding, "_here", lambda stream=None: (-1, 0))
    monkeypatch.setattr(mld.binding, "_lib", Library)

    def run(layout=1, has_bias=True, n=30, k=40, tokens=5, **change):
        plan = object.__new__(mld.FullyConnectedPlan)
        plan.desc, plan._h = mld.binding.FcDesc(n=n, k=k, weight_bits=8, has_bias=int(has_bias), dst_layout=layout, max_tokens=tokens), None
        plan._codes_sizes = mld.binding._codes_sizes(plan.desc)
        half, n4 = torch.float16, (n + 3) // 4 * 4
        t = dict(codes=torch.zeros(tokens, (k + 15) // 16 * 16, dtype=torch.int8), params=torch.zeros(tokens, 3),
                 weights=torch.zeros(n4 * k, dtype=torch.uint8), scale=torch.zeros(n, dtype=half), bias=torch.zeros(n4, dtype=half),
                 dst=torch.zeros(tokens, n if layout else n4, dtype=half))
        t.update(change)
        plan.run_codes(t["codes"], t["params"], t["weights"], t["scale"], t["dst"], tokens, bias=t["bias"])
        return calls.pop()

    return run


def test_what_fits_is_passed_on(call):
    assert call()[5] is not None and call(layout=0)[6] is not None
    assert call(has_bias=False, bias=None)[5] is None
    assert call(dst=torch.zeros(9, 30, dtype=torch.float16))[7] == 5


@pytest.mark.parametrize("name,tensor,words", [
    ("weights", torch.zeros(32 * 40 - 1, dtype=torch.uint8), "weights: expected at least 1280"),
    ("weights", torch.zeros(32 * 40, dtype=torch.float16), "weights: expected at least 1280"),
    ("weights", torch.zeros(32 * 40, 2, dtype=torch.uint8)[:, 0], "weights: expected at least 1280"),
    ("scale", torch.zeros(29, dtype=torch.float16), "scale: expected at least 30"), ("scale", torch.zeros(30), "scale: expected at least 30"),
    ("bias", torch.zeros(30, dtype=torch.float16), "bias: expected at least 32"), ("bias", torch.zeros(32), "bias: expected at least 32"),
    ("dst", torch.zeros(4, 30, dtype=torch.float16), "dst: expected at least 150"), ("dst", torch.zeros(5, 30), "dst: expected at least 150"),
    ("dst", torch.zeros(5, 60, dtype=torch.float16)[:, :30], "dst: expected at least 150"),
    ("codes", torch.zeros(5, 40, dtype=torch.int8), "codes: expected"), ("params", torch.zeros(5, 2), "params: expected")])
def test_what_does_not_fit_is_refused(call, name, tensor, words):
    with pytest.raises(ValueError, match=words):
        call(**{name: tensor})


def test_outputs_in_slices_are_whole_ones(call):
    with pytest.raises(ValueError, match="dst: expected at least 160"):
        call(layout=0, dst=torch.zeros(5, 30, dtype=torch.float16))


@pytest.mark.parametrize("name", ["codes", "params", "weights", "scale", "bias", "dst"])
def test_tensors_elsewhere_are_refused(call, mld, monkeypatch, name):
    monkeypatch.setattr(mld.binding, "_here", lambda stream=None: (-1, 0))
    shapes = dict(codes=(5, 48), params=(5, 3), weights=(1280,), scale=(30,), bias=(32,), dst=(5, 30))
    types = dict(codes=torch.int8, params=torch.float32, weights=torch.uint8)

    class Elsewhere(torch.Tensor):
        def get_device(self):
            return 1

    t = torch.zeros(shapes[name], dtype=types.get(name, torch.float16)).as_subclass(Elsewhere)
    with pytest.raises(ValueError, match=f"{name}: expected a tensor on the current GPU"):
        call(**{name: t})
