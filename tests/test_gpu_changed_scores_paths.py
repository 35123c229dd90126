"""The ways a program reaches biased_attention, tree_attention and commit_drafts (GPU): the native host path against
the general one, autograd's hooks and transforms, captured graphs, other streams, compiled models."""

import contextlib

import numpy as np
import pytest
import torch
import torch.utils.checkpoint

import sps_amd
from sps_amd import _native as N

pytestmark = pytest.mark.gpu


class _Off:
    biased_attention = tree_attention = staticmethod(lambda *a: None)
    commit_drafts = staticmethod(lambda *a: False)


@contextlib.contextmanager
def _general_path():
    real = N.binding()
    N._binding = _Off
    try:
        yield
    finally:
        N._binding = real


class _Counting:
    def __init__(self):
        self.real, self.taken = N.binding(), 0

    def __getattr__(self, name):
        def call(*args):
            r = getattr(self.real, name)(*args)
            self.taken += r is not None and r is not False
            return r
        return call

    def __enter__(self):
        N._binding = self
        return self

    def __exit__(self, *exc):
        N._binding = self.real


def _inputs(b=2, h=3, n=150, d=64, dtype=torch.bfloat16, layout="bnhd", seed=0):
    g = torch.Generator().manual_seed(seed)
    if layout == "packed":  # slices of one projection: strided, not dense
        p = torch.randn((b, n, 3, h, d), generator=g).to(dtype).cuda()
        ts = [p[:, :, i].transpose(1, 2) for i in range(3)]
    elif layout == "odd":  # rows not 16-byte aligned
        ts = [torch.randn((b, h, n, d + 1), generator=g).to(dtype).cuda()[..., :d] for _ in range(3)]
    else:
        ts = [torch.randn((b, n, h, d), generator=g).to(dtype).cuda().transpose(1, 2) for _ in range(3)]
    do = torch.randn((b, n, h, d), generator=g).to(dtype).cuda().transpose(1, 2)
    table = torch.randn((16, h), generator=g).to(dtype).cuda()
    slopes = torch.rand(h, generator=g).cuda()
    docs = (torch.arange(n, device="cuda") // 60).expand(b, n).contiguous()
    prefix = torch.arange(20, 20 + b, device="cuda", dtype=torch.int32)
    return ts, table, slopes, docs, prefix, do


def _call(ts, table, slopes, docs, prefix):
    return sps_amd.biased_attention(*ts, 0.125, softcap=4.0, slopes=slopes, bias_table=table, max_distance=50,
                                    documents_idx_BxT=docs, prefix_len_B=prefix)


@pytest.mark.parametrize("layout,taken", [("bnhd", 3), ("packed", 2), ("odd", 0)])
@pytest.mark.parametrize("form", ["all", "cap", "table", "slopes"])
def test_both_host_paths_agree(layout, taken, form):
    def both():
        ts, table, slopes, docs, prefix, do = _inputs(layout=layout, dtype=torch.float16 if form == "cap" else torch.bfloat16)
        leaves = [t.detach().requires_grad_() for t in ts]
        table = table.requires_grad_() if form in ("all", "table") else None
        kw = {"all": lambda: _call(leaves, table, slopes, docs, prefix),
              "cap": lambda: sps_amd.biased_attention(*leaves, 0.125, softcap=3),
              "table": lambda: sps_amd.biased_attention(*leaves, 0.125, bias_table=table, documents_idx_BxT=docs.int()),
              "slopes": lambda: sps_amd.biased_attention(*leaves, 0.125, slopes=slopes, prefix_len_B=prefix.long())}
        wrt = leaves + ([table] if table is not None else [])
        out = kw[form]()
        grads = torch.autograd.grad(out, wrt, do, retain_graph=True)
        again = torch.autograd.grad(out, wrt, do)
        with torch.no_grad():
            plain = kw[form]()
        with torch.inference_mode():
            inf = kw[form]()
        return [out, *grads, *again, plain, inf.clone()]

    with _Counting() as c:
        got = both()
        assert c.taken == taken
    with _general_path():
        want = both()
    for x, y in zip(got, want):
        assert torch.equal(x, y) and x.stride() == y.stride()


def test_partial_gradients():
    ts, table, slopes, docs, prefix, do = _inputs()
    full = None
    for wrt in ((0, 1, 2, 3), (0,), (2,), (3,), (1, 3)):
        res = []
        for ctx in (contextlib.nullcontext, _general_path):
            with ctx():
                leaves = [t.detach().requires_grad_(i in wrt) for i, t in enumerate((*ts, table))]
                o = _call(leaves[:3], leaves[3], slopes, docs, prefix)
                res.append(torch.autograd.grad(o, [leaves[i] for i in wrt], do))
        assert all(torch.equal(a, b) for a, b in zip(*res))
        full = full or res[0]
        assert all(torch.equal(full[i], x) for i, x in zip(wrt, res[0]))


def test_hooks_checkpoint_and_other_streams():
    ts, table, slopes, docs, prefix, do = _inputs()

    def grads(run):
        leaves = [t.detach().requires_grad_() for t in (*ts, table)]
        return torch.autograd.grad(run(*leaves), leaves, do)

    plain = lambda *x: _call(x[:3], x[3], slopes, docs, prefix)  # noqa: E731
    want = grads(plain)
    side = torch.cuda.Stream()

    def hooked(*x):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t):
            return plain(*x)

    def offloaded(*x):
        with torch.autograd.graph.save_on_cpu():
            return plain(*x)

    def on_stream(*x):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            o = plain(*x)
        torch.cuda.current_stream().wait_stream(side)
        o.record_stream(torch.cuda.current_stream())
        return o

    for run in (hooked, offloaded, on_stream,
                lambda *x: torch.utils.checkpoint.checkpoint(plain, *x, use_reentrant=False)):
        got = grads(run)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_transforms_agree_on_both_paths():
    ts, table, slopes, docs, prefix, do = _inputs(b=1, h=2, n=64)
    loss = lambda a, b, c, t: (_call((a, b, c), t, slopes, docs, prefix) * do).float().sum()  # noqa: E731
    res = []
    for ctx in (contextlib.nullcontext, _general_path):
        with ctx():
            leaves = [t.detach().requires_grad_() for t in (*ts, table)]
            out = _call(leaves[:3], leaves[3], slopes, docs, prefix)
            kinds = []
            for f in (lambda: torch.func.grad(loss, argnums=(0, 1, 2, 3))(*ts, table),
                      lambda: torch.autograd.grad(out, leaves, torch.stack([do, do * 2]), is_grads_batched=True,
                                                  retain_graph=True),
                      lambda: torch.autograd.grad(torch.autograd.grad(out, leaves, do, create_graph=True)[0].float().sum(),
                                                  leaves, retain_graph=True),
                      lambda: torch.vmap(lambda x: _call((x, x, x), table, slopes, docs, prefix))(torch.stack(ts[:2]))):
                try:
                    r = f()
                    kinds.append([t.clone() for t in (r if isinstance(r, tuple) else (r,))])
                except (RuntimeError, NotImplementedError) as e:
                    kinds.append(type(e).__name__)
            res.append(kinds)
    for a, b in zip(*res):
        assert a == b if isinstance(a, str) or isinstance(b, str) else all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_captured_training_step_replays():
    ts, table, slopes, docs, prefix, do = _inputs()
    leaves = [t.detach().requires_grad_() for t in (*ts, table)]

    def step():
        o = _call(leaves[:3], leaves[3], slopes, docs, prefix)
        return [o, *torch.autograd.grad(o, leaves, do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(4):
        fresh = _inputs(seed=seed + 1)
        with torch.no_grad():
            for t, x in zip((*leaves, do), (*fresh[0], fresh[1], fresh[5])):
                t.copy_(x)
            prefix.fill_(10 * seed)
        graph.replay()
        got = [t.clone() for t in outs]
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_compiled_models_trace_it():
    torch._dynamo.reset()
    ts, table, slopes, docs, prefix, do = _inputs()

    def model(q, k, v, t):
        return (_call((q, k, v), t, slopes, docs, prefix).float() * do).sum()

    res = []
    for fn in (model, torch.compile(model, fullgraph=True, backend="aot_eager")):
        leaves = [t.detach().clone().requires_grad_() for t in (*ts, table)]
        loss = fn(*leaves)
        res.append((loss.detach(), *torch.autograd.grad(loss, leaves)))
    assert all(torch.equal(x, y) for x, y in zip(*res))
    with torch.no_grad():
        one = torch.compile(lambda x: sps_amd.biased_attention(x, x, x, 0.1, softcap=2.0), fullgraph=True, backend="aot_eager")
        assert torch.equal(one(ts[0]), sps_amd.biased_attention(ts[0], ts[0], ts[0], 0.1, softcap=2.0))


def test_refusals_are_the_same_on_both_paths():
    ts, table, slopes, docs, prefix, _ = _inputs()
    q, k, v = ts
    b = sps_amd.biased_attention
    bad = [lambda: b(q, k, v, 0.1, softcap=-1.0), lambda: b(q, k, v, 0.1, softcap=float("nan")),
           lambda: b(q, k, v, 0.1, slopes=slopes.double()), lambda: b(q, k, v, 0.1, slopes=slopes[:2]),
           lambda: b(q, k, v, 0.1, slopes=slopes.cpu()), lambda: b(q, k, v, 0.1, slopes=slopes.clone().requires_grad_()),
           lambda: b(q, k, v, 0.1, bias_table=table[:, :2]), lambda: b(q, k, v, 0.1, bias_table=table, max_distance=8),
           lambda: b(q, k, v, 0.1, bias_table=table, max_distance=513), lambda: b(q, k, v, 0.1, bias_table=table[:1]),
           lambda: b(q, k, v, 0.1, bias_table=table.double()), lambda: b(q, k, v, 0.1, bias_table=table.cpu()),
           lambda: b(q, k, v, 0.1, prefix_len_B=prefix.float()), lambda: b(q, k, v, 0.1, prefix_len_B=prefix[:1]),
           lambda: b(q, k, v, 0.1, prefix_len_B=prefix.cpu()), lambda: b(q, k, v, 0.1, documents_idx_BxT=docs[:, :10]),
           lambda: b(q, k, v, float("inf")), lambda: b(q.float(), k.float(), v.float(), 0.1), lambda: b(q, k[:, :2], v, 0.1),
           lambda: b(q[..., :48], k[..., :48], v[..., :48], 0.1)]
    for f in bad:
        errors = []
        for ctx in (contextlib.nullcontext, _general_path):
            with ctx():
                with pytest.raises(Exception) as e:
                    f()
                errors.append((e.type, str(e.value)))
        assert errors[0] == errors[1]


# Draft trees ------------------------------------------------------------------------------------------------


def _tree(seed=0, b=3, t=6, h=2, d=64, storage=200, dtype=torch.bfloat16, index=torch.int64):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g).to(dtype).cuda()  # noqa: E731
    ln = torch.randint(0, storage - t, (b, h), generator=g).to(index).cuda()
    parents = torch.tensor([[-1, 0, 0, 1, 1, 4]] * b, dtype=index).cuda()[:, :t]
    return dict(q=r(b, t, h, d), dk=r(b, t, h, d), dv=r(b, t, h, d), k=r(b, h, storage, d), v=r(b, h, storage, d), len=ln,
                parents=parents, last=torch.tensor([5, -1, 3], dtype=index).cuda(), slopes=torch.rand(h, generator=g).cuda(),
                table=torch.randn((8, h), generator=g).cuda())


def _verify(s, **kw):
    seg = sps_amd.KVSegment(s["k"], s["v"], s["len"])
    o = sps_amd.tree_attention(s["q"], [seg], draft_k_BxTxHxD=s["dk"], draft_v_BxTxHxD=s["dv"], parents_BxT=s["parents"],
                               softcap=4.0, slopes=s["slopes"], bias_table=s["table"], max_distance=20, **kw)
    sps_amd.commit_drafts(seg, s["dk"], s["dv"], s["last"], parents_BxT=s["parents"])
    return [o, s["k"], s["v"], s["len"]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_tree_host_paths_agree(dtype, index):
    with _Counting() as c:
        got = [_verify(_tree(dtype=dtype, index=index)), _verify(_tree(dtype=dtype, index=index), sm_scale=0.3)]
        assert c.taken == 4
    with _general_path():
        want = [_verify(_tree(dtype=dtype, index=index)), _verify(_tree(dtype=dtype, index=index), sm_scale=0.3)]
    for x, y in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(x, y))


def test_a_captured_verification_step_replays():
    s = _tree()
    start = {x: s[x].clone() for x in ("k", "v", "len")}

    def restore():
        for x in start:
            s[x].copy_(start[x])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _verify(s)
    torch.cuda.current_stream().wait_stream(side)
    restore()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _verify(s)[0]
    for seed in range(4):
        fresh = _tree(seed + 1)
        for x in ("q", "dk", "dv"):
            s[x].copy_(fresh[x])
        s["last"].copy_(torch.tensor([seed, 5, -1]))
        restore()
        graph.replay()
        got = [t.clone() for t in (out, s["k"], s["v"], s["len"])]
        torch.cuda.synchronize()
        restore()
        want = _verify(s)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_calls_on_two_streams_at_once():
    # Every call has a workspace of its own.
    many = [_tree(i, storage=4000) for i in range(8)]
    for s in many:
        s["len"].fill_(3900)
    want = [[t.clone() for t in _verify({k: v.clone() for k, v in s.items()})] for s in many]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for i, s in enumerate(many):
        with torch.cuda.stream(streams[i % 4]):
            got.append(_verify(s))
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(x, y))


@pytest.mark.parametrize("leaf", ["q", "dk", "dv", "k", "v", "table"])
def test_tree_needs_no_grad(leaf):
    s = _tree()
    s[leaf].requires_grad_()
    for ctx in (contextlib.nullcontext, _general_path):
        with ctx():
            with pytest.raises(RuntimeError, match="no backward"):
                _verify(s)
            with torch.no_grad():
                _verify(s)


def test_tree_in_a_compiled_function():
    torch._dynamo.reset()
    s = _tree()
    want = _verify({k: v.clone() for k, v in s.items()})
    fn = torch.compile(lambda x: _verify(x)[0] * 2, backend="aot_eager")
    with torch.no_grad():
        got = fn(s)
    assert torch.equal(got, want[0] * 2) and torch.equal(s["k"], want[1]) and torch.equal(s["len"], want[3])


def test_tree_refusals_are_the_same_on_both_paths():
    s = _tree()
    seg = lambda **kw: sps_amd.KVSegment(**{"k": s["k"], "v": s["v"], "lengths": s["len"], **kw})  # noqa: E731
    t = lambda q=s["q"], segs=None, dk=s["dk"], dv=s["dv"], **kw: sps_amd.tree_attention(  # noqa: E731
        q, [seg()] if segs is None else segs, draft_k_BxTxHxD=dk, draft_v_BxTxHxD=dv, **kw)
    c = lambda g=None, dk=s["dk"], last=s["last"], **kw: sps_amd.commit_drafts(  # noqa: E731
        seg() if g is None else g, dk, s["dv"], last, **kw)
    big = torch.zeros((3, 65, 2, 64), device="cuda", dtype=torch.bfloat16)
    bad = [lambda: t(q=s["q"].float()), lambda: t(dk=s["dk"].half()), lambda: t(dk=s["dk"][:, :3]), lambda: t(dv=s["dv"].cpu()),
           lambda: t(q=big, dk=big, dv=big), lambda: t(segs=[seg()] * 4), lambda: t(segs=[seg(k=s["k"].half())]),
           lambda: t(segs=[seg(v=s["v"][:, :, :5])]), lambda: t(segs=[seg(lengths=s["len"].float())]),
           lambda: t(segs=[seg(lengths=s["len"][:2])]), lambda: t(segs=[seg(lengths=s["len"].cpu())]),
           lambda: t(segs=[seg(max_len_cap=-1)]), lambda: t(parents_BxT=s["parents"][:, :2]),
           lambda: t(parents_BxT=s["parents"].float()), lambda: t(parents_BxT=s["parents"].cpu()),
           lambda: t(softcap=0.0), lambda: t(bias_table=s["table"], max_distance=4), lambda: t(sm_scale=float("nan")),
           lambda: t(q=s["q"][..., :40], dk=s["dk"][..., :40], dv=s["dv"][..., :40]),
           lambda: t(segs=[seg(k=s["k"][..., 1:], v=s["v"][..., 1:])]),
           lambda: c(last=s["last"][:2]), lambda: c(last=s["last"].float()), lambda: c(last=s["last"].cpu()), lambda: c(dk=big),
           lambda: c(seg(lengths=s["len"][:, :1].expand(3, 2))), lambda: c(seg(k=s["k"][:, :1].expand_as(s["k"]))),
           lambda: c(seg(v=s["k"])), lambda: c(dk=s["k"].transpose(1, 2)[:, :6]), lambda: t(softcap=1e-20),
           lambda: t(sm_scale=1e35), lambda: c(dk=s["dk"].half()), lambda: c(seg(lengths=s["len"].float())), lambda: c(parents_BxT=s["parents"][:1])]
    for f in bad:
        errors = []
        for ctx in (contextlib.nullcontext, _general_path):
            with ctx():
                with pytest.raises(Exception) as e:
                    f()
                errors.append((e.type, str(e.value)))
        assert errors[0] == errors[1], errors


@pytest.mark.parametrize("length", [2 ** 63 - 1, 2 ** 63 - 3, -2 ** 63, 2 ** 31 + 5])
def test_lengths_no_cache_has(length):
    s, want = _tree(), _tree()
    s["len"].fill_(length)
    want["len"].fill_(200 if length > 0 else 0)
    k = s["k"].clone()
    got, full = _verify(s), _verify(want)[0]
    assert torch.equal(got[0], full) and torch.equal(s["k"], k) and (s["len"] == length).all()


def test_packed_caches_are_written_in_place():
    # Keys and values interleaved in one buffer, lengths a column of a wider table.
    s, p = _tree(), _tree()
    kv = torch.stack([p["k"], p["v"]], dim=3)
    p["k"], p["v"] = kv[:, :, :, 0], kv[:, :, :, 1]
    wide = torch.zeros((3, 2, 3), dtype=torch.int64, device="cuda")
    wide[:, :, 1] = p["len"]
    p["len"] = wide[:, :, 1]
    for ctx in (contextlib.nullcontext, _general_path):
        with ctx():
            assert all(torch.equal(a, b) for a, b in zip(_verify(s), _verify(p)))
    assert (wide[:, :, 0] == 0).all() and (wide[:, :, 2] == 0).all()


def test_python_tuples_of_segments_and_no_segments():
    s = _tree()
    seg = sps_amd.KVSegment(s["k"], s["v"], s["len"])
    kw = dict(draft_k_BxTxHxD=s["dk"], draft_v_BxTxHxD=s["dv"], parents_BxT=s["parents"])
    assert torch.equal(sps_amd.tree_attention(s["q"], (seg,), **kw), sps_amd.tree_attention(s["q"], [seg], **kw))
    none = sps_amd.KVSegment(s["k"], s["v"], torch.zeros_like(s["len"]))
    assert torch.equal(sps_amd.tree_attention(s["q"], [], **kw), sps_amd.tree_attention(s["q"], [none], **kw))


def test_drafts_of_uneven_batches():
    # Fewer drafts in some sequences: their rows past the last are padding, whatever they hold.
    s = _tree()
    want = _verify({k: v.clone() for k, v in s.items()})[0]
    s["parents"][1, 3:] = -2
    for x in ("q", "dk", "dv"):
        s[x][1, 3:] = float("nan")
    got = _verify(s)[0]
    assert torch.equal(got[[0, 2]], want[[0, 2]]) and torch.equal(got[1, :3], want[1, :3]) and (got[1, 3:] == 0).all()
    assert np.isfinite(got.float().cpu().numpy()).all()
