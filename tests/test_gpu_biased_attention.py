"""biased_attention (capped and biased scores, documents, prefixes) against the float64 oracle, forward and backward.

Every result is held, element by element, to the bound that oracle/biased.py derives from the kernels' roundings."""

import numpy as np
import pytest
import torch

import sps_amd
from oracle import biased as Bi

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
UNITS = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


def _docs(kind, b, n, r):
    if kind is None:
        return None
    if kind == "packed":
        return np.sort(r.integers(0, max(1, n // 40) + 2, (b, n)), axis=1)
    if kind == "single":
        return np.zeros((b, n), np.int64)
    if kind == "own":  # every position a document of its own
        return np.arange(n)[None].repeat(b, 0)
    return r.integers(0, 3, (b, n))  # ids that come back


class Case:
    def __init__(self, seed, b, h, n, d, dtype="bf16", cap=None, slopes=False, buckets=0, max_distance=128, docs=None,
                 prefix=None, table_dtype=None, gain=1.5, scale=None, hide=(), layout="bnhd"):
        r = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.table_dtype = dtype, table_dtype or dtype

        def rows(k):
            x = (torch.randn((b, n, h, d), generator=g) * k).to(DTYPES[dtype])
            return x.transpose(1, 2) if layout == "bnhd" else x.transpose(1, 2).contiguous()

        self.q, self.k, self.v, self.do = rows(gain), rows(gain), rows(1.0), rows(1.0)
        self.scale = d ** -0.5 if scale is None else scale
        self.cap, self.max_distance = cap, max_distance
        self.slopes = torch.tensor([2.0 ** (-8 * (i + 1) / h) for i in range(h)]) if slopes else None
        self.table = None
        if buckets:
            self.table = torch.randn((buckets, h), generator=g).to(DTYPES[self.table_dtype])
            for j in hide:
                self.table[j] = torch.finfo(self.table.dtype).min if j % 2 else -float("inf")
        self.docs = _docs(docs, b, n, r)
        self.prefix = None if prefix is None else np.array([prefix] * b if np.isscalar(prefix) else prefix)

    def leaves(self, device="cuda"):
        ts = [self.q, self.k, self.v] + ([self.table] if self.table is not None else [])
        out = []
        for t in ts:
            x = t.to(device, copy=True)
            assert x.stride() == t.stride()
            out.append(x.requires_grad_())
        return out

    def call(self, leaves, docs_dtype=torch.int64, prefix_dtype=torch.int32):
        docs = None if self.docs is None else torch.tensor(self.docs, device="cuda", dtype=docs_dtype)
        prefix = None if self.prefix is None else torch.tensor(self.prefix, device="cuda", dtype=prefix_dtype)
        return sps_amd.biased_attention(
            *leaves[:3], self.scale, softcap=self.cap, slopes=None if self.slopes is None else self.slopes.cuda(),
            bias_table=leaves[3] if len(leaves) > 3 else None, max_distance=self.max_distance, documents_idx_BxT=docs,
            prefix_len_B=prefix)

    def oracle(self):
        n = self.q.shape[2]
        see = Bi.visible(n, self.docs, None if self.prefix is None else np.clip(self.prefix, 0, n))
        q, k, v = (t.double().numpy() for t in (self.q, self.k, self.v))
        return Bi.Attention(q, k, v, self.scale, see, self.cap, None if self.slopes is None else self.slopes.numpy(),
                            None if self.table is None else self.table.double().numpy(), self.max_distance)


def _within(got, want, bound, what):
    got = got.detach().double().cpu().numpy()
    assert got.shape == want.shape and np.isfinite(got).all(), what
    off = np.abs(got - want) - bound
    i = np.unravel_index(np.argmax(off), off.shape) if off.size else None
    assert off.size == 0 or off[i] <= 0, f"{what}[{i}]: {got[i]} against {want[i]}, bound {bound[i]}"


def check(case, **call):
    ref = case.oracle()
    leaves = case.leaves()
    o = case.call(leaves, **call)
    _within(o, ref.o, ref.forward_bound(case.dtype), "o")
    grads = torch.autograd.grad(o, leaves, case.do.cuda())
    ref.backward(case.do.double().numpy())
    wants = [ref.dq, ref.dk, ref.dv] + ([ref.dtable] if ref.dtable is not None else [])
    for name, got, want, bound in zip(("dq", "dk", "dv", "dtable"), grads, wants,
                                      ref.backward_bounds(case.dtype, UNITS[case.table_dtype])):
        assert got.dtype == (case.q.dtype if name != "dtable" else case.table.dtype)
        _within(got, want, bound, name)
    with torch.no_grad():
        assert torch.equal(case.call(leaves, **call), o)


@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("change", [dict(cap=5.0), dict(slopes=True), dict(buckets=32), dict(cap=5.0, slopes=True),
                                    dict(cap=5.0, slopes=True, buckets=20, max_distance=65)])
def test_head_dims_and_changes(d, dtype, change):
    check(Case(1, 2, 3, 200, d, dtype, docs="packed", **change))


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 97, 128, 129, 257, 515])
@pytest.mark.parametrize("change", [dict(cap=3.0), dict(cap=8.0, buckets=16, max_distance=40, slopes=True)])
def test_lengths(n, change):
    check(Case(n, 2, 2, n, 64, **change))
    check(Case(n + 1, 1, 2, n, 128, docs="packed", prefix=n // 3, **change))


@pytest.mark.parametrize("docs", [None, "packed", "single", "own", "mixed"])
@pytest.mark.parametrize("prefix", [0, -5, 1, 40, 133, 100000, [7, 250]])
@pytest.mark.parametrize("d", [64, 128])
def test_documents_and_prefixes(docs, prefix, d):
    check(Case(3, 2, 2, 270, d, cap=6.0, slopes=True, buckets=32, docs=docs, prefix=prefix),
          docs_dtype=torch.int32, prefix_dtype=torch.int64)


@pytest.mark.parametrize("prefix", [None, 33])
def test_prefix_alone_and_nothing(prefix):
    check(Case(4, 2, 2, 150, 64, prefix=prefix))
    check(Case(5, 1, 2, 150, 32, "f16", prefix=prefix, docs="mixed"))


@pytest.mark.parametrize("buckets,top", [(2, 2), (2, 512), (3, 65), (16, 9), (32, 128), (64, 512), (200, 300),
                                         (256, 512), (255, 400)])
@pytest.mark.parametrize("table_dtype", ["bf16", "f32"])
def test_bucket_sizes(buckets, top, table_dtype):
    check(Case(6, 1, 3, 700, 64, buckets=buckets, max_distance=top, table_dtype=table_dtype))


@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_hidden_entries(d):
    # Distance 0 and two runs of distances hidden: the first rows see nothing and yield 0.
    c = Case(7, 1, 2, 160, d, cap=4.0, buckets=16, max_distance=60, hide=(0, 3, 9), table_dtype="f32")
    check(c)
    assert (c.call(c.leaves())[:, :, 0] == 0).all()


def test_every_entry_hidden():
    c = Case(8, 1, 2, 100, 64, slopes=True, buckets=4, max_distance=16, hide=(0, 1, 2, 3))
    leaves = c.leaves()
    o = c.call(leaves)
    assert (o == 0).all()
    for g in torch.autograd.grad(o, leaves, c.do.cuda()):
        assert (g == 0).all()


@pytest.mark.parametrize("scale,cap,gain", [(0.0, 2.0, 1.0), (-0.2, 2.0, 1.0), (0.125, 0.01, 1.0), (1.0, 80.0, 4.0),
                                            (0.125, 1e6, 1.0), (0.25, None, 3.0)])
def test_scales_and_caps(scale, cap, gain):
    check(Case(9, 1, 2, 190, 64, cap=cap, slopes=True, scale=scale, gain=gain))


def test_products_past_the_caps_range():
    # Products whose exponential overflows or vanishes: the cap's two limits, and no gradient from them.
    c = Case(10, 1, 1, 64, 64, cap=2.0, gain=40.0, scale=1.0)
    check(c)


@pytest.mark.parametrize("layout", ["bnhd", "bhnd"])
def test_layouts_and_slices(layout):
    check(Case(11, 2, 3, 140, 64, cap=5.0, buckets=32, layout=layout))
    base = torch.randn((2, 130, 3, 4, 64), device="cuda", dtype=torch.bfloat16)
    q, k, v = (x.transpose(1, 2) for x in base.unbind(2))
    odd = torch.randn((2, 4, 130, 65), device="cuda", dtype=torch.bfloat16)[..., 1:]  # unaligned rows: copied
    kw = dict(softcap=3.0, slopes=torch.rand(4, device="cuda"))
    for a in ((q, k, v), (odd, k, v), (q, odd, odd)):
        a = [t.detach().requires_grad_() for t in a]
        b = [t.detach().contiguous().requires_grad_() for t in a]
        oa, ob = sps_amd.biased_attention(*a, 0.125, **kw), sps_amd.biased_attention(*b, 0.125, **kw)
        assert torch.equal(oa, ob)
        do = torch.randn_like(ob)
        for x, y in zip(torch.autograd.grad(oa, a, do), torch.autograd.grad(ob, b, do)):
            assert torch.equal(x, y)


def test_table_views_and_strided_small_tensors():
    c = Case(12, 2, 3, 150, 64, cap=5.0, slopes=True, buckets=32, docs="packed", prefix=[3, 70])
    leaves = [t.detach() for t in c.leaves()]
    want = c.call(leaves)
    table = c.table.cuda().t().contiguous().t()  # bucket stride 1
    wide = torch.zeros((3, 2), device="cuda")
    wide[:, 0] = c.slopes.cuda()
    prefix = torch.zeros((2, 3), device="cuda", dtype=torch.int64)
    prefix[:, 1] = torch.tensor(c.prefix)
    got = sps_amd.biased_attention(*leaves[:3], c.scale, softcap=5.0, slopes=wide[:, 0], bias_table=table,
                                   documents_idx_BxT=torch.tensor(c.docs, device="cuda"), prefix_len_B=prefix[:, 1])
    assert torch.equal(got, want)


@pytest.mark.parametrize("shape", [(0, 2, 64, 64), (2, 0, 64, 64), (2, 2, 0, 64)])
def test_empty(shape):
    q, k, v = (torch.zeros(shape, device="cuda", dtype=torch.bfloat16, requires_grad=True) for _ in range(3))
    table = torch.zeros((8, shape[1]), device="cuda", requires_grad=True)
    o = sps_amd.biased_attention(q, k, v, 1.0, softcap=1.0, bias_table=table)
    assert o.shape == shape
    for g in torch.autograd.grad(o.float().sum(), [q, k, v, table]):
        assert (g == 0).all()


def test_only_the_table_learns_and_second_backward():
    c = Case(13, 2, 2, 300, 64, cap=5.0, buckets=32, docs="packed")
    leaves = c.leaves()
    for t in leaves[:3]:
        t.requires_grad_(False)
    o = c.call(leaves)
    a, = torch.autograd.grad(o, [leaves[3]], c.do.cuda(), retain_graph=True)
    b, = torch.autograd.grad(o, [leaves[3]], c.do.cuda())
    full = c.leaves()
    want = torch.autograd.grad(c.call(full), full, c.do.cuda())[3]
    assert torch.equal(a, b) and torch.equal(a, want)


def test_results_do_not_depend_on_timing():
    c = Case(14, 4, 6, 900, 64, cap=5.0, slopes=True, buckets=32, docs="packed", prefix=200)
    leaves, do = c.leaves(), c.do.cuda()
    first = None
    for _ in range(6):
        o = c.call(leaves)
        out = [o.detach(), *torch.autograd.grad(o, leaves, do)]
        first = first or out
        assert all(torch.equal(x, y) for x, y in zip(first, out))


def test_plain_full_attention_is_met():
    q, k, v = (torch.randn((2, 4, 400, 64), device="cuda", dtype=torch.bfloat16) for _ in range(3))
    zero = torch.zeros((2, 4), device="cuda")
    a = sps_amd.full_attention(q, k, v, 0.125)
    b = sps_amd.biased_attention(q, k, v, 0.125, bias_table=zero, max_distance=2)
    torch.testing.assert_close(a.float(), b.float(), atol=2 ** -7, rtol=2 ** -7)  # two roundings of P and O each


def test_random_cases():
    r = np.random.default_rng(2024)
    for i in range(24):
        buckets = int(r.choice([0, 0, 8, 32, 50]))
        n = int(r.integers(1, 420))
        c = dict(b=int(r.integers(1, 4)), h=int(r.integers(1, 4)), n=n, d=int(r.choice([16, 32, 64, 128, 256])),
                 dtype=str(r.choice(["bf16", "f16"])), cap=[None, 2.0, 30.0][r.integers(3)], slopes=bool(r.integers(2)),
                 buckets=buckets, max_distance=int(r.integers(buckets // 2 + 1, 513)),
                 docs=[None, "packed", "mixed"][r.integers(3)], prefix=[None, int(r.integers(0, n + 1))][r.integers(2)],
                 table_dtype=[None, "f32"][r.integers(2)])
        print("case", i, c, flush=True)
        check(Case(100 + i, **c))
