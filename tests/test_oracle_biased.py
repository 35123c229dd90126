"""The float64 oracle of attention with changed scores: against the document-masked oracle where nothing is changed,
against finite differences, and its bucket rule against the library's."""

import numpy as np
import pytest

import sps_amd
from oracle import attention as A
from oracle import biased as Bi
from oracle import mask as M


def _inputs(seed, b=2, h=2, n=24, d=8):
    r = np.random.default_rng(seed)
    return [r.standard_normal((b, h, n, d)) for _ in range(4)]


def test_unchanged_scores_equal_the_full_family():
    q, k, v, do = _inputs(0)
    docs = np.repeat([[0, 0, 0, 1, 1, 2]], 4, axis=1).reshape(1, -1).repeat(2, 0)
    docs.sort(axis=1)
    mask = M.batch_mask(M.FAMILY_FULL, docs)
    want, _ = A.forward(q, k, v, mask, 0.3)
    a = Bi.Attention(q, k, v, 0.3, Bi.visible(24, docs))
    np.testing.assert_allclose(a.o, want, atol=1e-12)
    a.backward(do)
    for got, ref in zip((a.dq, a.dk, a.dv), A.backward(q, k, v, do, mask, 0.3)):
        np.testing.assert_allclose(got, ref, atol=1e-12)


@pytest.mark.parametrize("which", ["q", "k", "v", "table"])
def test_gradients_against_differences(which):
    r = np.random.default_rng(1)
    q, k, v, do = _inputs(2)
    table, slopes = r.standard_normal((6, 2)), r.random(2)
    see = Bi.visible(24, prefix=[5, 17])

    def loss(x):
        args = {"q": q, "k": k, "v": v, "table": table, which: x}
        a = Bi.Attention(args["q"], args["k"], args["v"], 0.8, see, 2.0, slopes, args["table"], 12)
        return (a.o * do).sum()

    a = Bi.Attention(q, k, v, 0.8, see, 2.0, slopes, table, 12)
    a.backward(do)
    x = {"q": q, "k": k, "v": v, "table": table}[which]
    got = {"q": a.dq, "k": a.dk, "v": a.dv, "table": a.dtable}[which]
    for flat in r.choice(x.size, 12, replace=False):
        i = np.unravel_index(flat, x.shape)
        assert abs(Bi.finite_difference(loss, x, i) - got[i]) < 1e-6 * max(1.0, abs(got[i]))


def test_hidden_entries_and_empty_rows():
    q, k, v, _ = _inputs(3)
    table = np.zeros((2, 2))
    table[0, 0] = -3e38  # head 0: distance 0 hidden
    a = Bi.Attention(q, k, v, 1.0, Bi.visible(24), table=table, max_distance=8)
    assert (a.o[:, 0, 0] == 0).all() and (a.o[:, 1, 0] == v[:, 1, 0]).all()
    np.testing.assert_allclose(a.o[:, 0, 1], v[:, 0, 0])


@pytest.mark.parametrize("buckets", [2, 3, 7, 16, 32, 33, 48, 64, 128, 255, 256])
def test_buckets_of_the_library(buckets):
    for top in sorted({buckets // 2 + 1, buckets // 2 + 2, buckets, 2 * buckets, 128, 200, 256, 512}):
        if buckets // 2 < top <= 512:
            got = sps_amd.bias_buckets(600, buckets, top).tolist()
            assert got == [Bi.bucket(n, buckets, top) for n in range(600)], (buckets, top)


@pytest.mark.parametrize("buckets,top", [(1, 128), (257, 512), (32, 16), (32, 513), (-4, 128), (0, 128)])
def test_bucket_refusals(buckets, top):
    with pytest.raises(RuntimeError):
        sps_amd.bias_buckets(8, buckets, top)


def test_tree_helpers():
    see, depth = Bi.tree_see([-1, 0, 0, 1, -1, 9, 5, -2])
    assert depth.tolist() == [0, 1, 1, 2, 0, -1, -1, -1]
    assert see[3].nonzero()[0].tolist() == [0, 1, 3] and not see[5:].any()
    assert Bi.tree_path([-1, 0, 0, 1], 3) == [0, 1, 3]
    assert Bi.tree_path([-1, 0, 0, 1], -1) == [] == Bi.tree_path([-1, 9], 1)
