"""tree_attention at both sides of the rule by which one workgroup takes all keys of a row (GPU)."""

import pytest
import torch

import sps_amd
from test_gpu_tree_attention import Tree

pytestmark = pytest.mark.gpu

CHANGE = dict(cap=6.0, slopes=True, buckets=24, max_distance=90)


@pytest.mark.parametrize("scan", [511, 512, 513])
@pytest.mark.parametrize("t,d,dtype", [(1, 64, "bf16"), (7, 16, "f16"), (33, 128, "bf16"), (64, 256, "bf16"), (64, 32, "f16")])
@pytest.mark.parametrize("parents", ["tree", "padded"])
def test_few_rows(scan, t, d, dtype, parents):
    Tree(31, 2, 2, d, t, [scan], [[scan, 40]], dtype, parents=parents, **CHANGE).check()
    Tree(32, 2, 2, d, t, [0, scan], [[0, 0], [scan - 1, 0]], dtype, parents=parents).check()


@pytest.mark.parametrize("b,h", [(4, 32), (8, 32)])
@pytest.mark.parametrize("scan", [1024, 1025, 2048, 2049])
@pytest.mark.parametrize("t", [1, 9, 40])
def test_many_rows(b, h, scan, t):
    lengths = torch.linspace(0, scan, b).long()
    Tree(33, b, h, 16, t, [scan], [lengths], parents="padded", **CHANGE).check()


@pytest.mark.parametrize("t", [1, 12])
def test_one_segment_or_two(t):
    # The same keys in one segment (whole rows) and in two (chunks and their merge).
    g = torch.Generator().manual_seed(34)
    rnd = lambda *s: torch.randn(s, generator=g).bfloat16().cuda()  # noqa: E731
    q, dk, dv, k, v = rnd(2, t, 3, 64), rnd(2, t, 3, 64), rnd(2, t, 3, 64), rnd(2, 3, 480, 64), rnd(2, 3, 480, 64)
    seg = lambda x, y, n: sps_amd.KVSegment(x, y, torch.full((2,), n, device="cuda"))  # noqa: E731
    kw = dict(draft_k_BxTxHxD=dk, draft_v_BxTxHxD=dv, softcap=5.0, slopes=torch.rand(3, device="cuda"))
    one = sps_amd.tree_attention(q, [seg(k, v, 470)], **kw)
    two = sps_amd.tree_attention(q, [seg(k[:, :, :200], v[:, :, :200], 200), seg(k[:, :, 200:], v[:, :, 200:], 270)], **kw)
    # Both off the exact value by the rounding of P and of the result, 2^-8 each, of values up to 4.
    torch.testing.assert_close(one.float(), two.float(), rtol=4 * 2 ** -8, atol=2 * 2 ** -8 * 4)


def test_rows_too_far_apart_for_one_workgroup():
    # 400 keys 8 MiB apart: a row of them passes the 32-bit offsets that one workgroup's loads have.
    s, step, d = 400, 1 << 22, 64
    buf = torch.zeros(s * step, device="cuda", dtype=torch.bfloat16)
    k, v = (buf.as_strided((1, 1, s, d), (0, 0, step, 1), i * d) for i in range(2))
    k.copy_(torch.randn(k.shape, device="cuda"))
    v.copy_(torch.randn(v.shape, device="cuda"))
    q, dk, dv = torch.randn((3, 1, 5, 1, d), device="cuda").bfloat16()
    kw = dict(draft_k_BxTxHxD=dk, draft_v_BxTxHxD=dv)
    ln = torch.tensor([390], device="cuda")
    far = sps_amd.tree_attention(q, [sps_amd.KVSegment(k, v, ln)], **kw)
    near = sps_amd.tree_attention(q, [sps_amd.KVSegment(k.contiguous(), v.contiguous(), ln)], **kw)
    torch.testing.assert_close(far.float(), near.float(), rtol=4 * 2 ** -8, atol=2 * 2 ** -8 * 4)
