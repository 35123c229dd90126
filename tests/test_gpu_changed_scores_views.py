"""biased_attention on shared and broadcast inputs (GPU): keys and values of several heads, one table for all heads, one
prefix for the batch; each against the same call on copies."""

import pytest
import torch

import sps_amd

pytestmark = pytest.mark.gpu


def _inputs(b, h, kv, n, d, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(b * n + d)
    r = lambda *s: torch.randn(s, generator=g).to(dtype).cuda()  # noqa: E731
    q, k, v, do = r(b, n, h, d).transpose(1, 2), r(b, kv, n, d), r(b, kv, n, d), r(b, n, h, d).transpose(1, 2)
    return q, k, v, do, torch.randn((20, 1), generator=g).cuda(), (torch.arange(n, device="cuda") // 50)[None]


@pytest.mark.parametrize("b,h,n,d", [(2, 4, 150, 64), (1, 6, 300, 128), (4, 80, 130, 32)])
def test_shared_heads_and_broadcasts(b, h, n, d):
    kv = 2
    q, k, v, do, table, ids = _inputs(b, h, kv, n, d)

    def run(share):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, table)]
        lq, lk, lv, lt = leaves
        heads = [t[:, :, None].expand(b, kv, h // kv, n, d) for t in (lk, lv)]
        if share:
            wide = heads[0][:, 0], heads[1][:, 1]  # stride 0 over the heads
            wide = [w.expand(b, h // kv, n, d) for w in wide]
            args = (lq[:, :h // kv], *wide, d ** -0.5)
            docs, bias = ids.repeat(b, 1), lt.expand(20, h // kv)
            with pytest.raises(AssertionError):  # (as full_attention: document ids are dense)
                sps_amd.biased_attention(*args, documents_idx_BxT=ids.expand(b, n)[:, ::1] if b > 1 else ids.repeat(2, 1).T)
            prefix = torch.tensor([40], device="cuda").expand(b)
        else:
            args = (lq[:, :h // kv], heads[0][:, 0].contiguous(), heads[1][:, 1].contiguous(), d ** -0.5)
            docs, bias, prefix = ids.repeat(b, 1), lt.repeat(1, h // kv), torch.full((b,), 40, device="cuda")
        o = sps_amd.biased_attention(*args, softcap=5.0, bias_table=bias, max_distance=60, documents_idx_BxT=docs,
                                     prefix_len_B=prefix)
        return [o, *torch.autograd.grad(o, leaves, do[:, :h // kv])]

    shared, copied = run(True), run(False)
    for x, y in zip(shared, copied):
        assert torch.equal(x, y)
    assert (shared[2][:, 1] == 0).all() and shared[2][:, 0].abs().sum() > 0
