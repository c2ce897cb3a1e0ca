"""Calls of the norm that the binding refuses, without a GPU."""
import pytest
import torch


def test_codes_and_params_go_together(monkeypatch):
    import __graft_entry__ as g
    g.build()
    mld = g.import_package()
    monkeypatch.setattr(mld.binding, "_here", lambda stream=None: (-1, 0))
    x = torch.zeros(3, 64, dtype=torch.float16)
    for alone in (dict(codes=torch.zeros(3, 64, dtype=torch.int8)), dict(params=torch.zeros(3, 3))):
        with pytest.raises(ValueError, match="codes and params go together"):
            mld.add_rms_norm(x, out=torch.empty_like(x), **alone)


def test_a_batch_without_tokens_is_no_error(monkeypatch):
    """Empty tensors have no address."""
    import __graft_entry__ as g
    g.build()
    mld = g.import_package()
    monkeypatch.setattr(mld.binding, "_here", lambda stream=None: (-1, 0))
    x = torch.zeros(0, 64, dtype=torch.float16)
    codes, params = torch.zeros(0, 64, dtype=torch.int8), torch.zeros(0, 3)
    mld.add_rms_norm(x, out=torch.empty_like(x), codes=codes, params=params)
    mld.add_rms_norm(x, residual=x, sum_out=torch.empty_like(x), out=torch.empty_like(x))
    mld.MoeRouter(64, 2).run(x, torch.zeros(0, 2, dtype=torch.int32), torch.zeros(0, 2))
