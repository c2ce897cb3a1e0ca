"""Calls of the norm, the router and the experts that the host refuses, without a GPU: nothing of them reaches a kernel."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def mld():
    import __graft_entry__ as g
    g.build()
    return g.import_package()


def _norm_io(mld, **change):
    io = mld.binding.AddNormIo(1 << 20, 64, 2 << 20, 64, 3 << 20, 4 << 20, 64, 5 << 20, 64, 6 << 20, 64, 7 << 20)
    for name, value in change.items():
        setattr(io, name, value)
    return io


@pytest.mark.parametrize("desc,change,words", [
    (dict(width=0), {}, b"width"), (dict(width=16385), {}, b"width"), (dict(eps=-1.0), {}, b"eps"), (dict(eps=float("nan")), {}, b"eps"),
    (dict(weight_offset=float("inf")), {}, b"weight_offset"), ({}, dict(out=None, codes=None, params=None), b"neither"),
    ({}, dict(params=None), b"params"), ({}, dict(residual=None), b"residual"), ({}, dict(x=None), b"null"),
    ({}, dict(x=(1 << 20) + 1), b"aligned"), ({}, dict(x_stride=-64), b"stride"), ({}, dict(out_stride=63), b"stride"),
    ({}, dict(sum_stride=0), b"stride"), ({}, dict(out=1 << 20, out_stride=128), b"stride"),
    ({}, dict(sum_out=2 << 20, residual_stride=72), b"stride"), ({}, dict(out=4 << 20), b"same"), ({}, dict(codes=(6 << 20) + 8), b"16-byte"),
    ({}, dict(codes_stride=48), b"codes"), ({}, dict(codes_stride=72), b"codes")])
def test_norm(mld, desc, change, words):
    d = mld.binding.AddNormDesc(64, 1e-6, 0.0, 1, 0)
    for name, value in desc.items():
        setattr(d, name, value)
    assert mld.lib().mld_add_rms_norm(ctypes.byref(d), ctypes.byref(_norm_io(mld, **change)), 2, None) == mld.INVALID_ARGUMENT
    assert words in mld.lib().mld_last_error()
    if desc or change.get("codes", 1) is None:
        return
    assert mld.lib().mld_add_rms_norm(ctypes.byref(mld.binding.AddNormDesc(64, 1e-6, 0.0, 1, 0)), ctypes.byref(_norm_io(mld)), 0, None) == mld.OK


@pytest.mark.parametrize("change,words", [
    (dict(experts=0), b"experts"), (dict(experts=1025), b"experts"), (dict(top_k=0), b"top_k"), (dict(top_k=33), b"top_k"),
    (dict(score=2), b"score"), (dict(groups=3), b"groups"), (dict(groups=64, top_groups=64), b"groups"), (dict(groups=8, top_groups=9), b"top_groups"),
    (dict(groups=8, top_groups=1, top_k=9), b"top_k"), (dict(group_best=3), b"group_best"), (dict(groups=32, top_groups=32, experts=32, group_best=2), b"group_best"),
    (dict(factor=float("nan")), b"factor")])
def test_router(mld, change, words):
    d = mld.binding.MoeRouteDesc(64, 8, 0, 1, 1, 1, 1, 1.0, 1)
    for name, value in change.items():
        setattr(d, name, value)
    run = mld.lib().mld_moe_route
    assert run(ctypes.byref(d), 1 << 20, 64, None, 2 << 20, 3 << 20, 1, None) == mld.INVALID_ARGUMENT
    assert words in mld.lib().mld_last_error()
    d = mld.binding.MoeRouteDesc(64, 8, 0, 1, 1, 1, 1, 1.0, 1)
    assert run(ctypes.byref(d), None, 64, None, 2 << 20, 3 << 20, 1, None) == mld.INVALID_ARGUMENT
    assert run(ctypes.byref(d), 1 << 20, -64, None, 2 << 20, 3 << 20, 1, None) == mld.INVALID_ARGUMENT
    assert run(ctypes.byref(d), (1 << 20) + 1, 64, None, 2 << 20, 3 << 20, 1, None) == mld.INVALID_ARGUMENT
    assert run(ctypes.byref(d), 1 << 20, 64, (4 << 20) + 2, 2 << 20, 3 << 20, 1, None) == mld.INVALID_ARGUMENT
    assert run(ctypes.byref(d), None, 64, None, None, None, 0, None) == mld.OK


@pytest.mark.parametrize("change,words", [
    (dict(experts=0), b"experts"), (dict(experts=1025), b"experts"), (dict(top_k=33), b"top_k"), (dict(d_model=48), b"d_model"),
    (dict(ffn=32800), b"d_model"), (dict(ffn=0), b"d_model"), (dict(weight_bits=2), b"WeightsDescription"), (dict(block=16), b"block"),
    (dict(d_model=96, block=64), b"block"), (dict(activation=2), b"activation"), (dict(max_tokens=0), b"max_tokens"),
    (dict(max_tokens=65537), b"max_tokens"), (dict(force_path=3), b"force_path")])
def test_experts(mld, change, words):
    d = mld.binding.MoeDesc(4, 2, 128, 64, 4, 32, 0, 8, -1, 0)
    for name, value in change.items():
        setattr(d, name, value)
    h = ctypes.c_void_p()
    assert mld.lib().mld_moe_plan_create(ctypes.byref(d), ctypes.byref(h)) == mld.INVALID_ARGUMENT and not h
    assert words in mld.lib().mld_last_error()


def test_null_plans(mld):
    lib = mld.lib()
    assert lib.mld_moe_plan_create(None, None) == mld.INVALID_ARGUMENT
    assert lib.mld_moe_run(None, None, 1, None) == mld.INVALID_ARGUMENT
    assert lib.mld_moe_plan_destroy(None) == mld.OK and lib.mld_moe_plan_workspace_bytes(None) == 0
    assert lib.mld_moe_plan_device_status(None, None) == mld.INVALID_ARGUMENT
    assert lib.mld_fc_run_codes(None, None, None, None, None, None, None, 1, None) == mld.INVALID_ARGUMENT


def test_tensors_in_host_memory_and_of_other_shapes_are_refused(mld):
    import torch
    x = torch.zeros(3, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="x: expected a tensor on the current GPU, got one on cpu"):
        mld.add_rms_norm(x, out=torch.empty_like(x))
    with pytest.raises(ValueError, match="expected float16 or float32"):
        mld.add_rms_norm(x.double(), out=x.double())
    with pytest.raises(ValueError, match="logits: expected a tensor on the current GPU"):
        mld.MoeRouter(64, 2).run(x, torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2))
