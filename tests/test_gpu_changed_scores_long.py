"""biased_attention on long rows of many heads (GPU): tiles of 128 with far, near and ahead blocks; a few heads against the
float64 oracle, which sees each head alone."""

import copy

import pytest
import torch

from test_gpu_biased_attention import UNITS, Case, _within

pytestmark = pytest.mark.gpu


def check_heads(case, heads):
    leaves = case.leaves()
    o = case.call(leaves)
    grads = torch.autograd.grad(o, leaves, case.do.cuda())
    sub = copy.copy(case)
    sub.q, sub.k, sub.v, sub.do = (t[:, heads] for t in (case.q, case.k, case.v, case.do))
    sub.slopes = case.slopes[heads] if case.slopes is not None else None
    sub.table = case.table[:, heads] if case.table is not None else None
    ref = sub.oracle()
    _within(o[:, heads], ref.o, ref.forward_bound(case.dtype), "o")
    ref.backward(sub.do.double().numpy())
    bounds = ref.backward_bounds(case.dtype, UNITS[case.table_dtype])
    for name, got, want, bound in zip(("dq", "dk", "dv"), grads, (ref.dq, ref.dk, ref.dv), bounds):
        _within(got[:, heads], want, bound, name)
    if case.table is not None:
        _within(grads[3][:, heads], ref.dtable, bounds[3], "dtable")


@pytest.mark.parametrize("d,dtype", [(32, "bf16"), (64, "bf16"), (64, "f16"), (128, "bf16"), (256, "bf16")])
@pytest.mark.parametrize("change", [dict(cap=8.0), dict(buckets=32), dict(cap=8.0, slopes=True, buckets=40, max_distance=300)])
@pytest.mark.parametrize("docs,prefix", [(None, None), ("packed", 700), ("single", 300)])
def test_long_rows_of_many_heads(d, dtype, change, docs, prefix):
    check_heads(Case(41, 1, 33, 1030, d, dtype, docs=docs, prefix=prefix, gain=1.0, **change), [0, 17, 32])
