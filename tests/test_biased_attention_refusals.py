"""What biased_attention and its C entry points refuse, before anything reaches a GPU."""

import ctypes as C

import pytest
import torch

import sps_amd
from sps_amd import _native as N
from sps_amd.biased_attention import check_change


def test_cpu_tensors_are_refused():
    q = torch.zeros((1, 2, 8, 64), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU"):
        sps_amd.biased_attention(q, q, q, 1.0, softcap=1.0)


@pytest.mark.parametrize("cap", [0.0, -1.0, float("nan"), float("inf")])
def test_caps(cap):
    with pytest.raises(ValueError, match="softcap"):
        check_change(cap, None, None, 128, 2, torch.device("cpu"))


def test_slopes():
    cpu = torch.device("cpu")
    with pytest.raises(TypeError, match="slopes"):
        check_change(None, torch.zeros(2, dtype=torch.float64), None, 128, 2, cpu)
    with pytest.raises(ValueError, match="slopes"):
        check_change(None, torch.zeros(3), None, 128, 2, cpu)
    with pytest.raises(ValueError, match="no gradient"):
        check_change(None, torch.zeros(2, requires_grad=True), None, 128, 2, cpu)
    with pytest.raises(ValueError, match="slopes"):
        check_change(None, torch.zeros(2), None, 128, 2, torch.device("meta"))


@pytest.mark.parametrize("shape,dtype,top,error", [
    ((32, 3), torch.float32, 128, ValueError), ((32,), torch.float32, 128, ValueError),
    ((1, 2), torch.float32, 128, ValueError), ((257, 2), torch.float32, 512, ValueError),
    ((32, 2), torch.float32, 16, ValueError), ((32, 2), torch.float32, 513, ValueError),
    ((32, 2), torch.float64, 128, TypeError)])
def test_tables(shape, dtype, top, error):
    with pytest.raises(error):
        check_change(None, None, torch.zeros(shape, dtype=dtype), top, 2, torch.device("cpu"))


def _gpu():
    return torch.cuda.is_available()


def _call(backward=False, change=None, **over):
    a = dict(B=1, H=2, N=64, D=64, dtype=N.DTYPE_BF16, ptr=0x10000, strides=(8192, 4096, 64), docs=None,
             docs_dtype=N.DTYPE_I64, prefix=None, prefix_dtype=N.DTYPE_I32, scale=0.125, dtable=None, ws=0x40000,
             ws_bytes=1 << 20)
    a.update(over)
    c = N.ScoreChange(softcap=1.0) if change is None else change
    st, p = N.i64_array(a["strides"]), a["ptr"]
    head = (a["B"], a["H"], a["N"], a["D"], a["dtype"])
    tail = (a["docs"], a["docs_dtype"], 64, a["prefix"], a["prefix_dtype"], a["scale"], C.byref(c) if c else None)
    if backward:
        return N.lib().sps_biased_bwd(*head, *(p, st) * 5, 0x20000, *(p, st) * 3, a["dtable"], *tail, 0, a["ws"],
                                      a["ws_bytes"], None)
    return N.lib().sps_biased_fwd(*head, *(p, st) * 4, 0x20000, *tail, a["ws"], a["ws_bytes"], None)


def _change(**over):
    c = N.ScoreChange(softcap=0.0, bias_table=0x30000, table_dtype=N.DTYPE_F32, num_buckets=32, max_distance=128)
    for k, v in over.items():
        setattr(c, k, v)
    return c


@pytest.mark.skipif(_gpu(), reason="fake device addresses: CPU build only")
@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("over,code,needle", [
    (dict(D=48), N.SPS_E_UNSUPPORTED, "head_dim"), (dict(dtype=N.DTYPE_F32), N.SPS_E_UNSUPPORTED, "dtype"),
    (dict(ptr=0x10008), N.SPS_E_INVALID, "aligned"), (dict(ptr=0), N.SPS_E_INVALID, "null"),
    (dict(strides=(8192, 4096, 60)), N.SPS_E_INVALID, "multiple of 8"), (dict(scale=float("nan")), N.SPS_E_INVALID, "sm_scale"),
    (dict(docs=0x50000, docs_dtype=N.DTYPE_F32), N.SPS_E_INVALID, "document ids"),
    (dict(docs=0x50000, ws_bytes=0), N.SPS_E_WORKSPACE, "workspace"),
    (dict(prefix=0x50000, prefix_dtype=N.DTYPE_F32), N.SPS_E_INVALID, "prefix_len"),
    (dict(change=False), N.SPS_E_INVALID, "change"), (dict(N=-1), N.SPS_E_INVALID, "negative"),
    (dict(change=N.ScoreChange(softcap=-1.0)), N.SPS_E_INVALID, "softcap"),
    (dict(change=N.ScoreChange(softcap=float("inf"))), N.SPS_E_INVALID, "softcap"),
    (dict(change=_change(table_dtype=N.DTYPE_I32)), N.SPS_E_UNSUPPORTED, "table dtype"),
    (dict(change=_change(num_buckets=1)), N.SPS_E_UNSUPPORTED, "num_buckets"),
    (dict(change=_change(num_buckets=300)), N.SPS_E_UNSUPPORTED, "num_buckets"),
    (dict(change=_change(max_distance=16)), N.SPS_E_UNSUPPORTED, "max_distance"),
    (dict(change=_change(max_distance=1000)), N.SPS_E_UNSUPPORTED, "max_distance")])
def test_c_abi(backward, over, code, needle):
    assert _call(backward, **over) == code and needle in N.last_error()


@pytest.mark.skipif(_gpu(), reason="fake device addresses: CPU build only")
def test_c_abi_backward_only():
    assert _call(True, dtable=0x60000) == N.SPS_E_INVALID and "dtable" in N.last_error()
    need = N.lib().sps_biased_workspace_bytes(1, 2, 64, 0, 1, 32)
    assert need > N.lib().sps_biased_workspace_bytes(1, 2, 64, 0, 1, 0) > 0
    assert _call(True, change=_change(), dtable=0x60000, ws_bytes=need - 1) == N.SPS_E_WORKSPACE
    assert _call(False, B=0) == N.SPS_OK and _call(True, N=0) == N.SPS_OK


def test_workspace_sizes():
    f = N.lib().sps_biased_workspace_bytes
    assert f(2, 4, 300, 0, 0, 0) == 0 and f(-1, 4, 300, 0, 1, 0) == 0
    assert f(2, 4, 300, 1, 1, 32) >= f(2, 4, 300, 1, 1, 0) + 2 * 4 * 3 * 32 * 4
