"""Calls of biased_attention, tree_attention and commit_drafts that must be refused before anything runs (CPU: the C
entries with addresses that no kernel reads)."""

import ctypes as C

import pytest
import torch

from sps_amd import _native as N
from sps_amd.biased_attention import check_change

cpu_only = pytest.mark.skipif(torch.cuda.is_available(), reason="fake device addresses: CPU build only")
CPU = torch.device("cpu")


@pytest.mark.parametrize("cap", [2.0 ** -11, 1e-45, 2.0 ** 21, 1e38, 1e39, 10 ** 400])
def test_caps_past_fp32(cap):
    with pytest.raises(ValueError, match="softcap"):
        check_change(cap, None, None, 128, 2, CPU)
    if cap < 1e39:
        st, change = N.i64_array((8192, 4096, 64)), N.ScoreChange(softcap=cap)
        assert N.lib().sps_biased_fwd(1, 2, 64, 64, N.DTYPE_BF16, *(0x10000, st) * 4, 0x20000, None, 0, 0, None, N.DTYPE_I32,
                                      1.0, C.byref(change), None, 0, None) == N.SPS_E_INVALID
        assert "softcap" in N.last_error()


def test_caps_at_the_limits():
    assert check_change(2.0 ** -10, None, None, 128, 2, CPU) == 2.0 ** -10
    assert check_change(2 ** 20, None, None, 128, 2, CPU) == 2.0 ** 20


@cpu_only
@pytest.mark.parametrize("scale", [1e31, -1e31, 3e38])
def test_scales_past_fp32(scale):
    st, change = N.i64_array((8192, 4096, 64)), N.ScoreChange(softcap=1.0)
    assert N.lib().sps_biased_fwd(1, 2, 64, 64, N.DTYPE_BF16, *(0x10000, st) * 4, 0x20000, None, 0, 0, None, N.DTYPE_I32,
                                  scale, C.byref(change), None, 0, None) == N.SPS_E_INVALID
    assert "sm_scale" in N.last_error()


def _commit(b=2, h=2, t=4, d=64, k=0x100000, v=0x200000, k_st=(8192, 4096, 64), v_st=(8192, 4096, 64), storage=64,
            per_head=1, len_st=(2, 1), dk=0x300000, dv=0x400000, draft_st=(512, 128, 64)):
    ds = N.i64_array(draft_st)
    return N.lib().sps_commit_drafts(b, h, d, t, N.DTYPE_BF16, k, v, N.i64_array((*k_st, *v_st)), storage, 0x500000,
                                     N.DTYPE_I64, per_head, N.i64_array(len_st), dk, ds, dv, ds, None, N.DTYPE_I32, t,
                                     0x600000, N.DTYPE_I64, None)


@cpu_only
@pytest.mark.parametrize("over,needle", [
    (dict(k_st=(0, 4096, 64)), "overlap"), (dict(v_st=(8192, 0, 64)), "overlap"), (dict(k_st=(8192, 4096, 0)), "overlap"),
    (dict(k_st=(8192, 4096, 56)), "overlap"), (dict(len_st=(0, 1)), "overlap"), (dict(len_st=(2, 0)), "overlap"),
    (dict(per_head=0, len_st=(0, 0)), "overlap"), (dict(v=0x100000), "share"),
    (dict(dk=0x100000), "drafts"), (dict(dv=0x200000 + 32768 - 16), "drafts"), (dict(dv=0x100000 - 1024), "drafts")])
def test_commit_onto_shared_memory(over, needle):
    assert _commit(**over) == N.SPS_E_INVALID and needle in N.last_error()



@cpu_only
def test_more_workgroups_than_a_launch_has():
    st, change = N.i64_array((0, 0, 64)), N.ScoreChange(softcap=1.0)
    assert N.lib().sps_biased_fwd(4096, 4096, 128, 64, N.DTYPE_BF16, *(0x10000, st) * 4, 0x20000, None, 0, 0, None, N.DTYPE_I32,
                                  1.0, C.byref(change), None, 0, None) == N.SPS_E_UNSUPPORTED
    assert "workgroups" in N.last_error()
    ds = N.i64_array((512, 128, 64))
    scan = N.i64_array([100])
    rows = N.i64_array((0, 0, 64))
    ptr, one = N.ptr_const((0x10000,)), N.i32_const((1,))
    assert N.lib().sps_tree_attention(4096, 4096, 64, 1, N.DTYPE_BF16, 0x10000, ds, 1, ptr, rows, ptr, rows, ptr,
                                      N.i32_const((N.DTYPE_I64,)), one, scan, 0x10000, ds, 0x10000, ds, None, N.DTYPE_I32, 1,
                                      1.0, None, 0x20000, 0x30000, 1 << 40, None) == N.SPS_E_UNSUPPORTED
    assert "workgroups" in N.last_error()
