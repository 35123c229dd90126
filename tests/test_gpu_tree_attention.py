"""tree_attention and commit_drafts against their oracles: trees, chains and single tokens, over every kind of cache."""

import numpy as np
import pytest
import torch

import sps_amd
from oracle import biased as Bi

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def random_parents(r, b, t, padding=0.0):
    p = np.array([[int(r.integers(-1, i)) if i else -1 for i in range(t)] for _ in range(b)])
    if padding:
        bad = r.random((b, t)) < padding
        p = np.where(bad, r.choice([-2, -7, t, 1000, 2 ** 31 - 1], (b, t)), p)
    return p


class Tree:
    def __init__(self, seed, b, h, d, t, storages, lengths, dtype="bf16", parents="tree", cap=None, slopes=False,
                 buckets=0, max_distance=128, gain=1.5, len_dtype=torch.int64, caps=None, junk=True, view=False,
                 parents_dtype=torch.int32, scale=None):
        r = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.cap, self.max_distance, self.scale = dtype, cap, max_distance, scale
        rnd = lambda *s, k=1.0: (torch.randn(s, generator=g) * k).to(DTYPES[dtype])  # noqa: E731
        self.q, self.dk, self.dv = rnd(b, t, h, d, k=gain), rnd(b, t, h, d, k=gain), rnd(b, t, h, d)
        self.segs = []
        for i, s in enumerate(storages):
            k, v = rnd(b, h, s, d, k=gain), rnd(b, h, s, d)
            ln = torch.as_tensor(lengths[i]).to(len_dtype)
            top = s if caps is None or caps[i] is None else max(1, min(s, caps[i])) if s else 0
            if junk:  # what lies past the live rows may be anything
                at = torch.arange(s)[None, None]
                dead = (at >= ln.reshape(b, -1, 1).clamp(max=top)).expand(b, h, s)
                k[dead], v[dead] = float("nan"), float("inf")
            self.segs.append((k, v, ln, None if caps is None else caps[i]))
        if parents == "chain":
            self.parents = None
        else:
            self.parents = random_parents(r, b, t, 0.25 if parents == "padded" else 0.0)
            if parents == "padded" and junk:
                for i in range(b):
                    none = torch.tensor(Bi.tree_see(list(self.parents[i]))[1] < 0)
                    self.dk[i, none], self.dv[i, none], self.q[i, none] = float("nan"), float("inf"), float("nan")
        self.parents_dtype = parents_dtype
        self.slopes = torch.tensor([2.0 ** (-8 * (i + 1) / h) for i in range(h)]) if slopes else None
        self.table = torch.randn((buckets, h), generator=g).to(DTYPES[dtype]) if buckets else None
        self.view = view

    def args(self):
        def dev(x):
            if self.view:  # [B, S, H, D] memory behind a [B, H, S, D] view, as a prefill leaves it
                return x.transpose(1, 2).contiguous().cuda().transpose(1, 2)
            return x.cuda()

        segs = [sps_amd.KVSegment(dev(k), dev(v), n.cuda(), max_len_cap=c) for k, v, n, c in self.segs]
        parents = None if self.parents is None else torch.tensor(self.parents, dtype=self.parents_dtype, device="cuda")
        return segs, dict(draft_k_BxTxHxD=self.dk.cuda(), draft_v_BxTxHxD=self.dv.cuda(), parents_BxT=parents,
                          sm_scale=self.scale, softcap=self.cap, slopes=None if self.slopes is None else self.slopes.cuda(),
                          bias_table=None if self.table is None else self.table.cuda(), max_distance=self.max_distance)

    def run(self):
        segs, kw = self.args()
        return sps_amd.tree_attention(self.q.cuda(), segs, **kw)

    def check(self, out=None):
        out = self.run() if out is None else out
        assert out.dtype == self.q.dtype and out.is_contiguous()
        b, t, h, d = self.q.shape
        scale = d ** -0.5 if self.scale is None else self.scale
        parents = self.parents if self.parents is not None else np.arange(-1, t - 1)[None].repeat(b, 0)
        clean = lambda x: torch.nan_to_num(x.double(), 0.0, 0.0, 0.0).numpy()  # noqa: E731  (dead rows: never used)
        segs = [(clean(k), clean(v), n.numpy(), None if c is None else max(1, c)) for k, v, n, c in self.segs]
        want, mag = Bi.tree_attend(clean(self.q), segs, clean(self.dk), clean(self.dv), parents, scale, self.cap,
                                   None if self.slopes is None else self.slopes.numpy(),
                                   None if self.table is None else self.table.double().numpy(), self.max_distance)
        # As oracle/biased.py derives: P rounded to the inputs' type (u), a weight off by twice the score's error, the
        # result rounded once (u); the partial records and their merge are fp32.
        u, tiny = (2.0 ** -8, 2.0 ** -126) if self.dtype == "bf16" else (2.0 ** -11, 2.0 ** -25)
        e = 2.0 ** -24
        raw = abs(scale) * max([np.abs(clean(self.q)).max() * np.abs(x).max() * d for x in
                                [clean(self.dk)] + [s[0] for s in segs if s[0].size]])
        past = sum(s[0].shape[2] for s in segs) + t
        big = raw + (self.cap or 0) + (float(self.slopes.max()) * past if self.slopes is not None else 0) + 8
        eps = 2 * ((d + 4) * e * raw + 8 * e * (self.cap or 0.0) + 8 * e * big + 32 * e)
        bound = (u + eps) * mag + u * np.abs(want) + tiny * (1 + past)
        got = out.double().cpu().numpy()
        assert np.isfinite(got).all()
        off = np.abs(got - want) - bound
        i = np.unravel_index(np.argmax(off), off.shape)
        assert off[i] <= 0, f"{i}: {got[i]} against {want[i]}, bound {bound[i]}"
        for i in range(b):
            for x in np.flatnonzero(Bi.tree_see(list(parents[i]))[1] < 0):
                assert (got[i, x] == 0).all()


@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("t", [1, 5, 32, 33, 64])
def test_head_dims_and_drafts(d, dtype, t):
    Tree(1, 2, 2, d, t, [300], [[257, 300]], dtype, cap=6.0 if t != 5 else None, slopes=t > 1, buckets=16 * (t % 2)).check()


@pytest.mark.parametrize("length", [0, 1, 31, 32, 33, 127, 128, 129, 255, 256, 511, 512, 513, 1000, -3, 5000])
@pytest.mark.parametrize("t,d", [(1, 64), (7, 64), (40, 128)])
def test_lengths(length, t, d):
    Tree(length + 7, 1, 2, d, t, [1000], [[length]], buckets=16, max_distance=40).check()


@pytest.mark.parametrize("storages,lengths,caps", [
    ([], [], None), ([0], [[0, 0]], None), ([64, 700], [[64, 9], [[700, 3], [0, 513]]], None),
    ([16, 130, 300], [[0, 16], [[130, 1], [77, 0]], [299, 4]], None), ([200, 0, 90], [[5, 200], [0, 0], [90, 17]], None),
    ([500, 300], [[500, 40], [300, 300]], [130, None]), ([500], [[500, 3]], [0])])
@pytest.mark.parametrize("change", [dict(), dict(cap=4.0, slopes=True, buckets=32, max_distance=200)])
def test_segments(storages, lengths, caps, change):
    for t in (1, 9, 50):
        Tree(t, 2, 2, 64, t, storages, lengths, caps=caps, len_dtype=torch.int32, **change).check()


@pytest.mark.parametrize("parents", ["tree", "chain", "padded"])
@pytest.mark.parametrize("parents_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("t", [1, 3, 31, 64])
def test_trees(parents, parents_dtype, t):
    Tree(t, 3, 2, 64, t, [150], [[150, 0, 33]], parents=parents, parents_dtype=parents_dtype, buckets=8,
         max_distance=10, slopes=True).check()
    Tree(t, 3, 1, 128, t, [150], [[150, 0, 33]], parents=parents, parents_dtype=parents_dtype).check()


def test_nothing_but_padding():
    x = Tree(3, 2, 2, 64, 6, [100], [[100, 50]], parents="padded")
    x.parents[:] = -2
    assert (x.run() == 0).all()


@pytest.mark.parametrize("change", [dict(), dict(cap=20.0), dict(buckets=32), dict(slopes=True), dict(cap=9.0, slopes=True, buckets=64, max_distance=512)])
def test_long_caches(change):
    Tree(5, 2, 2, 64, 4, [9000], [[9000, 6001]], **change).check()
    Tree(6, 1, 2, 128, 61, [5000], [[4999]], **change).check()


@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0])
def test_scales(scale):
    Tree(7, 2, 2, 64, 8, [300], [[300, 20]], cap=3.0, scale=scale).check()


def test_views_and_strided_drafts():
    x = Tree(8, 2, 3, 64, 6, [260, 40], [[[260, 3, 100], [9, 0, 260]], [40, 11]], buckets=16)
    want = x.run()
    x.check(want)
    x.view = True
    assert torch.equal(x.run(), want)
    segs, kw = x.args()
    packed = torch.stack([x.q, x.dk, x.dv], dim=2).cuda()  # [B, T, 3, H, D]
    kw["draft_k_BxTxHxD"], kw["draft_v_BxTxHxD"] = packed[:, :, 1], packed[:, :, 2]
    assert torch.equal(sps_amd.tree_attention(packed[:, :, 0], segs, **kw), want)
    odd = torch.zeros((2, 6, 3, 65), dtype=x.q.dtype, device="cuda")
    odd[..., 1:] = x.q.cuda()
    assert torch.equal(sps_amd.tree_attention(odd[..., 1:], segs, **kw), want)
    lens = torch.zeros((2, 3, 2), dtype=torch.int64, device="cuda")
    lens[..., 0] = x.segs[0][2].cuda()
    segs[0].lengths = lens[..., 0]
    assert torch.equal(sps_amd.tree_attention(x.q.cuda(), segs, **kw), want)


def test_offsets_past_32_bits():
    # One cache row every 2^19 elements: the 5000th key lies 5 GiB behind the first.
    s, step = 5000, 1 << 19
    pool = torch.empty((s * step,), dtype=torch.bfloat16, device="cuda")
    k = pool.as_strided((1, 1, s, 64), (s * step, s * step, step, 1))
    v = pool.as_strided((1, 1, s, 64), (s * step, s * step, step, 1), 128)
    x = Tree(9, 1, 1, 64, 3, [s], [[4990]])
    k.copy_(x.segs[0][0].cuda())
    v.copy_(x.segs[0][1].cuda())
    segs, kw = x.args()
    want = sps_amd.tree_attention(x.q.cuda(), segs, **kw)
    segs[0].k, segs[0].v = k, v
    assert torch.equal(sps_amd.tree_attention(x.q.cuda(), segs, **kw), want)
    draft = torch.randn((1, 3, 1, 64), device="cuda", dtype=torch.bfloat16)
    sps_amd.commit_drafts(segs[0], draft, draft, torch.tensor([2], device="cuda"))
    assert segs[0].lengths.tolist() == [4993] and torch.equal(k[0, 0, 4990:4993], draft[0, :, 0])


def test_empty_batch():
    q = torch.zeros((0, 4, 2, 64), device="cuda", dtype=torch.bfloat16)
    seg = sps_amd.KVSegment(*(torch.zeros((0, 2, 8, 64), device="cuda", dtype=torch.bfloat16) for _ in range(2)),
                            torch.zeros(0, device="cuda", dtype=torch.int64))
    assert sps_amd.tree_attention(q, [seg], draft_k_BxTxHxD=q, draft_v_BxTxHxD=q).shape == (0, 4, 2, 64)
    sps_amd.commit_drafts(seg, q, q, torch.zeros(0, device="cuda", dtype=torch.int64))


def test_one_token_is_the_decode_step():
    # Unchanged scores, one draft: masked_kv_attention with the token's own key as the extra one.
    x = Tree(10, 4, 4, 64, 1, [700], [[700, 1, 333, 0]], junk=False)
    segs, kw = x.args()
    want = sps_amd.masked_kv_attention(x.q[:, 0].cuda(), segs, attn_dtype=torch.bfloat16,
                                       extra_kv=[(kw["draft_k_BxTxHxD"][:, 0], kw["draft_v_BxTxHxD"][:, 0])])
    torch.testing.assert_close(x.run()[:, 0].float(), want, atol=2 ** -7, rtol=2 ** -7)


def test_random_trees():
    r = np.random.default_rng(77)
    for i in range(30):
        b, h, d = int(r.integers(1, 4)), int(r.integers(1, 4)), int(r.choice([16, 32, 64, 128, 256]))
        n = int(r.integers(0, 4))
        storages = [int(r.integers(0, 800)) for _ in range(n)]
        lengths = [r.integers(-2, s + 3, (b, h) if r.integers(2) else (b,)) for s in storages]
        buckets = int(r.choice([0, 0, 6, 32]))
        kw = dict(dtype=str(r.choice(["bf16", "f16"])), parents=str(r.choice(["tree", "chain", "padded"])),
                  cap=[None, 3.0, 30.0][r.integers(3)], slopes=bool(r.integers(2)), buckets=buckets,
                  max_distance=int(r.integers(buckets // 2 + 1, 300)), view=bool(r.integers(2)))
        t = int(r.integers(1, 65))
        print("case", i, b, h, d, t, storages, kw, flush=True)
        Tree(200 + i, b, h, d, t, storages, lengths, **kw).check()


# Commit ---------------------------------------------------------------------------------------------------


def commit_check(seed, b, h, d, t, storage, lengths, last, dtype="bf16", parents="tree", len_dtype=torch.int64,
                 index_dtype=torch.int64, view=False):
    r = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g).to(DTYPES[dtype])  # noqa: E731
    k, v, dk, dv = rnd(b, h, storage, d), rnd(b, h, storage, d), rnd(b, t, h, d), rnd(b, t, h, d)
    ln = torch.as_tensor(lengths).to(len_dtype)
    p = None if parents == "chain" else random_parents(r, b, t, 0.25 if parents == "padded" else 0.0)
    dev = (lambda x: x.transpose(1, 2).contiguous().cuda().transpose(1, 2)) if view else (lambda x: x.cuda())
    seg = sps_amd.KVSegment(dev(k), dev(v), ln.cuda())
    sps_amd.commit_drafts(seg, dk.cuda(), dv.cuda(), torch.tensor(last, device="cuda", dtype=index_dtype),
                          parents_BxT=None if p is None else torch.tensor(p, device="cuda", dtype=index_dtype))
    want = ln.clone()
    for i in range(b):
        path = Bi.tree_path(list(p[i]) if p is not None else list(range(-1, t - 1)), last[i])
        for j in range(h):
            n = int(ln[i, j] if ln.dim() == 2 else ln[i])
            if n < 0 or n >= storage:
                continue
            fit = path[:storage - n]
            k[i, j, n:n + len(fit)], v[i, j, n:n + len(fit)] = dk[i, fit, j], dv[i, fit, j]
            if ln.dim() == 2:
                want[i, j] = n + len(fit)
            else:
                want[i] = n + len(fit)
    assert torch.equal(seg.k.cpu(), k) and torch.equal(seg.v.cpu(), v) and torch.equal(seg.lengths.cpu(), want)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [16, 64, 256])
@pytest.mark.parametrize("parents", ["tree", "chain", "padded"])
def test_commit(dtype, d, parents):
    r = np.random.default_rng(d)
    for t in (1, 6, 64):
        last = r.integers(-1, t, 5).tolist()
        commit_check(t, 5, 3, d, t, 90, r.integers(0, 80, (5, 3)), last, dtype, parents)
        commit_check(t, 5, 3, d, t, 90, r.integers(0, 80, 5), last, dtype, parents, torch.int32, torch.int32, True)


@pytest.mark.parametrize("lengths", [[[0, 89], [90, 88], [-1, 200]], [86, 90, -4]])
def test_commit_at_the_end(lengths):
    commit_check(1, 3, 2, 64, 8, 90, lengths, [7, 7, 7], parents="chain")


@pytest.mark.parametrize("last", [-1, -100, 8, 10 ** 12])
def test_commit_of_no_draft(last):
    commit_check(2, 2, 2, 64, 8, 50, [[1, 2], [3, 4]], [last, 3])


def test_commit_many_heads_and_sequences():
    r = np.random.default_rng(9)
    commit_check(3, 70, 5, 64, 16, 64, r.integers(0, 64, (70, 5)), r.integers(-1, 16, 70).tolist())
    commit_check(4, 1, 600, 16, 9, 30, r.integers(0, 30, (1, 600)), [8], parents="chain")
    commit_check(5, 1, 33, 256, 64, 100, r.integers(0, 64, (1, 33)), [63], "f32", parents="chain")


# Together -------------------------------------------------------------------------------------------------


def _prefix_and_step(model, cap, slopes, table):
    """Reference: dense attention over a whole sequence's q, k, v [1, H, N, D]."""
    q, k, v = model
    return sps_amd.biased_attention(q, k, v, q.shape[-1] ** -0.5, softcap=cap, slopes=slopes, bias_table=table)


@pytest.mark.parametrize("change", [(None, False, 0), (5.0, True, 32)])
def test_prefill_verify_commit_and_go_on(change):
    """A prompt's prefill, then rounds of a drafted tree: verified, its best path committed, verified rows equal to
    the rows of one dense pass over the accepted tokens."""
    cap, use_slopes, buckets = change
    torch.manual_seed(5)
    h, d, n, storage = 4, 64, 90, 256
    slopes = torch.tensor([0.5, 0.25, 0.1, 0.02], device="cuda") if use_slopes else None
    table = torch.randn((buckets, h), device="cuda").bfloat16() if buckets else None
    new = lambda t: [torch.randn((1, h, t, d), device="cuda", dtype=torch.bfloat16) for _ in range(3)]  # noqa: E731
    seq = new(n)
    seg = sps_amd.KVSegment(*(torch.full((1, h, storage, d), float("nan"), device="cuda", dtype=torch.bfloat16)
                              for _ in range(2)), torch.tensor([n], device="cuda"))
    seg.k[:, :, :n], seg.v[:, :, :n] = seq[1], seq[2]
    r = np.random.default_rng(1)
    for t, last in ((8, 6), (1, 0), (40, 39), (5, -1), (3, 2)):
        draft = new(t)
        parents = random_parents(r, 1, t)
        out = sps_amd.tree_attention(draft[0].transpose(1, 2), [seg], draft_k_BxTxHxD=draft[1].transpose(1, 2),
                                     draft_v_BxTxHxD=draft[2].transpose(1, 2),
                                     parents_BxT=torch.tensor(parents, device="cuda"), softcap=cap, slopes=slopes,
                                     bias_table=table)
        sps_amd.commit_drafts(seg, draft[1].transpose(1, 2), draft[2].transpose(1, 2), torch.tensor([last], device="cuda"),
                              parents_BxT=torch.tensor(parents, device="cuda"))
        path = Bi.tree_path(list(parents[0]), last)
        if path:
            seq = [torch.cat([x, y[:, :, path]], dim=2) for x, y in zip(seq, draft)]
            dense = _prefix_and_step(seq, cap, slopes, table)[:, :, -len(path):]
            # Two kernels' roundings of P and of the result (2^-8 each) on outputs of magnitude up to ~4.
            torch.testing.assert_close(out[:, path].transpose(1, 2).float(), dense.float(), atol=4 * 2 ** -7, rtol=2 ** -7)
        assert seg.lengths.item() == seq[0].shape[2]
        assert torch.equal(seg.k[:, :, :seg.lengths.item()], seq[1])
