"""What tree_attention, commit_drafts and their C entry points refuse, before anything reaches a GPU."""

import ctypes as C

import pytest
import torch

import sps_amd
from sps_amd import _native as N

cpu_only = pytest.mark.skipif(torch.cuda.is_available(), reason="fake device addresses: CPU build only")


def test_cpu_tensors_are_refused():
    q = torch.zeros((1, 2, 2, 64), dtype=torch.bfloat16)
    kv = torch.zeros((1, 2, 8, 64), dtype=torch.bfloat16)
    seg = sps_amd.KVSegment(kv, kv.clone(), torch.zeros(1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="GPU"):
        sps_amd.tree_attention(q, [seg], draft_k_BxTxHxD=q, draft_v_BxTxHxD=q)
    with pytest.raises(RuntimeError, match="GPU"):
        sps_amd.commit_drafts(seg, q, q, torch.zeros(1, dtype=torch.int64))


def _tree(**over):
    a = dict(B=2, H=2, D=64, T=4, dtype=N.DTYPE_BF16, q=0x10000, strides=(512, 128, 64), n_seg=1, k=0x20000,
             ks=(16384, 8192, 64), v=0x30000, len=0x40000, len_dtype=N.DTYPE_I64, scan=128, draft=0x50000,
             ds=(512, 128, 64), parents=0x60000, parents_dtype=N.DTYPE_I32, scale=0.125, change=None, out=0x70000,
             ws=0x80000, ws_bytes=1 << 24)
    a.update(over)
    n = max(a["n_seg"], 1)
    st, ds, ks = N.i64_array(a["strides"]), N.i64_array(a["ds"]), N.i64_array(a["ks"] * n)
    change = C.byref(a["change"]) if a["change"] is not None else None
    return N.lib().sps_tree_attention(
        a["B"], a["H"], a["D"], a["T"], a["dtype"], a["q"], st, a["n_seg"], N.ptr_array([a["k"]] * n), ks,
        N.ptr_array([a["v"]] * n), ks, N.ptr_array([a["len"]] * n), N.i32_array([a["len_dtype"]] * n),
        N.i32_array([0] * n), N.i64_array([a["scan"]] * n), a["draft"], ds, a["draft"], ds, a["parents"],
        a["parents_dtype"], a["T"], a["scale"], change, a["out"], a["ws"], a["ws_bytes"], None)


@cpu_only
@pytest.mark.parametrize("over,code,needle", [
    (dict(T=0), N.SPS_E_UNSUPPORTED, "drafts"), (dict(T=65), N.SPS_E_UNSUPPORTED, "drafts"),
    (dict(D=80), N.SPS_E_UNSUPPORTED, "head_dim"), (dict(dtype=N.DTYPE_F32), N.SPS_E_UNSUPPORTED, "dtype"),
    (dict(B=-1), N.SPS_E_INVALID, "negative"), (dict(B=70000), N.SPS_E_UNSUPPORTED, "65535"),
    (dict(n_seg=4), N.SPS_E_INVALID, "segments"), (dict(scan=-1), N.SPS_E_INVALID, "scan"),
    (dict(scan=1 << 31), N.SPS_E_UNSUPPORTED, "2^30"), (dict(q=None), N.SPS_E_INVALID, "null"),
    (dict(q=0x10008), N.SPS_E_INVALID, "aligned"), (dict(strides=(512, 128, 60)), N.SPS_E_INVALID, "16 bytes"),
    (dict(k=None), N.SPS_E_INVALID, "null"), (dict(v=0x30004), N.SPS_E_INVALID, "aligned"),
    (dict(ks=(16384, 8192, 68)), N.SPS_E_INVALID, "16 bytes"), (dict(ks=(16384, 8192, -64)), N.SPS_E_INVALID, "negative"),
    (dict(ks=(16384, 8192, 1 << 24)), N.SPS_E_UNSUPPORTED, "stride too large"), (dict(len=None), N.SPS_E_INVALID, "null"),
    (dict(len_dtype=N.DTYPE_F32), N.SPS_E_INVALID, "lengths"), (dict(draft=None), N.SPS_E_INVALID, "null"),
    (dict(ds=(512, -128, 64)), N.SPS_E_INVALID, "negative"), (dict(parents_dtype=N.DTYPE_U8), N.SPS_E_INVALID, "parents"),
    (dict(scale=float("inf")), N.SPS_E_INVALID, "sm_scale"), (dict(out=None), N.SPS_E_INVALID, "out"),
    (dict(ws_bytes=100), N.SPS_E_WORKSPACE, "workspace"), (dict(ws=None), N.SPS_E_INVALID, "workspace"),
    (dict(change=N.ScoreChange(softcap=float("nan"))), N.SPS_E_INVALID, "softcap")])
def test_tree_abi(over, code, needle):
    assert _tree(**over) == code and needle in N.last_error()


@cpu_only
def test_empty_batches_are_no_work():
    assert _tree(B=0) == N.SPS_OK and _tree(H=0) == N.SPS_OK and _commit(B=0) == N.SPS_OK and _commit(storage=0) == N.SPS_OK


def test_a_workspace_serves_smaller_calls():
    # The library takes longer chunks where the records of its own choice would not fit.
    f = N.lib().sps_tree_workspace_bytes
    size = lambda b, scan, t=8: f(b, 4, 64, t, 1, N.i64_array([scan]))  # noqa: E731
    assert size(0, 100) >= 0 and size(2, -1) == 0 and size(2, 100, 65) == 0
    assert size(64, 8192) > 0
    records = lambda b, scan, chunk: b * 4 * (-(-scan // chunk) + 1) * 8 * 68 * 4  # noqa: E731
    for b, scan in ((1, 100), (8, 8192), (64, 300), (63, 8191)):
        assert min(records(b, scan, c) for c in (128, 256, 512, 1024, 2048, 4096)) <= size(64, 8192)


def _commit(**over):
    a = dict(B=2, H=2, D=64, T=4, dtype=N.DTYPE_BF16, k=0x10000, v=0x20000, strides=(8192, 4096, 64) * 2, storage=64,
             len=0x30000, len_dtype=N.DTYPE_I64, draft=0x40000, ds=(512, 128, 64), parents=None, parents_dtype=N.DTYPE_I32,
             last=0x50000, last_dtype=N.DTYPE_I64)
    a.update(over)
    ds = N.i64_array(a["ds"])
    return N.lib().sps_commit_drafts(a["B"], a["H"], a["D"], a["T"], a["dtype"], a["k"], a["v"],
                                     N.i64_array(a["strides"]), a["storage"], a["len"], a["len_dtype"], 1,
                                     N.i64_array([2, 1]), a["draft"], ds, a["draft"], ds, a["parents"],
                                     a["parents_dtype"], 4, a["last"], a["last_dtype"], None)


@cpu_only
@pytest.mark.parametrize("over,code,needle", [
    (dict(T=65), N.SPS_E_UNSUPPORTED, "drafts"), (dict(D=8), N.SPS_E_UNSUPPORTED, "head_dim"),
    (dict(dtype=N.DTYPE_I32), N.SPS_E_UNSUPPORTED, "dtype"), (dict(storage=-1), N.SPS_E_INVALID, "storage"),
    (dict(k=None), N.SPS_E_INVALID, "null"), (dict(v=0x20002), N.SPS_E_INVALID, "aligned"),
    (dict(strides=(8192, 4096, 65) * 2), N.SPS_E_INVALID, "16 bytes"), (dict(len=None), N.SPS_E_INVALID, "null"),
    (dict(len_dtype=N.DTYPE_F32), N.SPS_E_INVALID, "lengths"), (dict(draft=0x40001), N.SPS_E_INVALID, "aligned"),
    (dict(last=None), N.SPS_E_INVALID, "null"), (dict(last_dtype=N.DTYPE_U8), N.SPS_E_INVALID, "last"),
    (dict(parents=0x60000, parents_dtype=N.DTYPE_BF16), N.SPS_E_INVALID, "parents")])
def test_commit_abi(over, code, needle):
    assert _commit(**over) == code and needle in N.last_error()
