"""Calls around the 4-bit cache that the host refuses, without a GPU: nothing of them reaches a kernel."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def mld():
    import __graft_entry__ as g
    g.build()
    return g.import_package()


def _io(mld, **change):
    io = mld.binding.QkRopeIo()
    io.q, io.k, io.q_out, io.k_out, io.positions = 1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20
    io.q_stride = io.q_out_stride = 512
    io.k_stride = io.k_out_stride = 256
    for name, value in change.items():
        setattr(io, name, value)
    return io


@pytest.mark.parametrize("change", [dict(q_out_stride=0), dict(k_out_stride=0), dict(q_stride=0, q_out=1 << 20, q_out_stride=0),
                                    dict(q_out=1 << 20, q_out_stride=1024), dict(k_out=2 << 20, k_stride=512), dict(q_stride=-512),
                                    dict(k_out_stride=-256), dict(q_stride=256), dict(k_stride=8)])
def test_tokens_that_would_write_one_row_or_read_what_another_wrote_are_refused(mld, change):
    plan = mld.QkNormRope(4, 2, 128)
    io = _io(mld, **change)
    assert mld.lib().mld_qk_rope_run(plan._h, ctypes.byref(io), 2, None) == mld.INVALID_ARGUMENT
    assert b"stride" in mld.lib().mld_last_error()


def test_tensors_in_host_memory_are_refused(mld):
    import torch
    with pytest.raises(ValueError, match="GPU"):
        mld.Kv4Cache(2, 64, 16, 4, device="cpu")
    with pytest.raises(ValueError, match="GPU"):
        mld.Kv4Cache(2, 64, 16, 4, pool=torch.zeros(1, 4, 2, 1, 18 * 64, dtype=torch.uint8))
    q, k = torch.zeros(3, 4, 64, dtype=torch.float16), torch.zeros(3, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="q: expected a tensor on the current GPU, got one on cpu"):
        mld.QkNormRope(4, 2, 64).run(q, k, torch.zeros(3, dtype=torch.int32), torch.empty_like(q), torch.empty_like(k))
