"""biased_attention at both sides of the rules that choose a kernel's form by the number of tiles (GPU)."""

import pytest

from test_gpu_biased_attention import Case, check

pytestmark = pytest.mark.gpu

CHANGES = [dict(cap=5.0), dict(slopes=True), dict(buckets=32), dict(cap=5.0, slopes=True, buckets=20, max_distance=65)]


@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("change", CHANGES)
@pytest.mark.parametrize("docs,prefix", [(None, None), ("packed", None), ("mixed", 40), (None, 70)])
def test_many_tiles(d, change, docs, prefix):
    # 280 tiles: past every limit.
    check(Case(21, 4, 35, 135, d, "f16" if docs else "bf16", docs=docs, prefix=prefix, **change))


@pytest.mark.parametrize("b,h", [(1, 256), (1, 257), (2, 64), (3, 43), (8, 8), (5, 13)])
@pytest.mark.parametrize("d", [32, 128, 256])
def test_around_the_limits(b, h, d):
    check(Case(22, b, h, 67, d, cap=4.0, buckets=16, max_distance=30))


@pytest.mark.parametrize("n", [31, 32, 33, 64, 65, 96, 127, 129, 160])
@pytest.mark.parametrize("docs", [None, "packed", "mixed"])
def test_short_rows(n, docs):
    for d, change in ((64, CHANGES[0]), (128, CHANGES[3])):
        check(Case(n, 2, 2, n, d, docs=docs, prefix=n // 4, **change))
        check(Case(n, 2, 2, n, d, docs=docs, layout="bhnd", **change))


@pytest.mark.parametrize("d", [64, 128])
def test_long_rows_of_few_heads(d):
    for change in (CHANGES[0], CHANGES[3]):
        check(Case(23, 1, 1, 2100, d, gain=1.0, **change))
        check(Case(24, 1, 1, 2081, d, docs="packed", prefix=900, gain=1.0, **change))
