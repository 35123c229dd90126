"""biased_attention's torch.library registration (CPU: fake tensors, no kernel runs)."""

import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import sps_amd  # noqa: F401  (registers the ops)
from sps_amd import _native as N


def test_fake_impls_give_the_kernels_layouts():
    with FakeTensorMode():
        q = torch.empty(2, 64, 3, 32, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
        docs = torch.zeros(2, 64, dtype=torch.int64, device="cuda")
        table = torch.empty(16, 3, dtype=torch.float32, device="cuda")
        o, lse, ws = torch.ops.sps_amd.biased_attention_fwd(q, q, q, docs, None, None, table, 0.125, 5.0, 50, 16)
        assert o.shape == (2, 3, 64, 32) and o.transpose(1, 2).is_contiguous()
        assert lse.shape == (2, 3, 64) and lse.dtype == torch.float32
        assert ws.numel() == N.lib().sps_biased_workspace_bytes(2, 3, 64, 1, 1, 16)
        assert torch.ops.sps_amd.biased_attention_fwd(q, q, q, docs, None, None, table, 0.125, 5.0, 50, -1)[2].numel() == 0
        dq, dk, dv, dt = torch.ops.sps_amd.biased_attention_bwd(o, q, q, q, o, lse, docs, None, None, table, ws, 0.125, 5.0,
                                                                50, 16)
        assert dq.shape == q.shape and dq.stride() == q.stride() and dt.shape == (16, 3) and dt.dtype == torch.float32


def test_the_ops_are_pure():
    for op in (torch.ops.sps_amd.biased_attention_fwd, torch.ops.sps_amd.biased_attention_bwd):
        assert all(a.alias_info is None or not a.alias_info.is_write for a in op.default._schema.arguments)
