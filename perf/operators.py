"""Operators of sps_amd on attention with changed scores, and their plain forms, over the sizes programs call them at.

Four kinds of work:

* ``forward`` / ``train``: one layer of document-masked causal attention whose scores are capped by a tanh, lose a
  multiple of the distance or get a learned bias by distance buckets, with a prefix that every query sees; without
  gradients (prefill, evaluation) or with them (output and the gradients of q, k, v and the bias table);
* ``tree``: the tokens of a draft tree, or one token, of every sequence against the sequence's cached keys and the
  tokens' own ancestors, with the same score changes;
* ``commit``: the accepted path of each sequence's drafts appended to its cache.

Where ``own`` is false ``run`` takes the plain form, elementary torch operations in fp32; where it is true, the
package's public entry points. ``exact`` is the definition in float64.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
GAIN = 1.5            # of queries and keys: scores with a standard deviation of GAIN^2, so that a cap has work
MAX_FLOPS = 2.7e11    # no drawn case costs more than the largest listed ones
MAX_BYTES = 6.1e8


def _attn(name, kind, batch, heads, head_dim, tokens, *, cap=0.0, slopes=False, buckets=0, max_distance=128, docs=False,
          prefix=False, dtype="bf16"):
    return {"name": name, "kind": kind, "batch": batch, "heads": heads, "head_dim": head_dim, "tokens": tokens,
            "cap": cap, "slopes": slopes, "buckets": buckets, "max_distance": max_distance, "docs": docs,
            "prefix": prefix, "dtype": dtype}


def _cache(name, kind, batch, heads, head_dim, drafts, len_lo, len_hi, storage, *, ring=0, chain=False, cap=0.0,
           slopes=False, buckets=0, max_distance=128, dtype="bf16"):
    return {"name": name, "kind": kind, "batch": batch, "heads": heads, "head_dim": head_dim, "drafts": drafts,
            "len_lo": len_lo, "len_hi": len_hi, "storage": storage, "ring": ring, "chain": chain, "cap": cap,
            "slopes": slopes, "buckets": buckets, "max_distance": max_distance, "dtype": dtype}


def listed():
    return [
        # Evaluation of short rows with capped scores: the smallest call, where the launch counts.
        _attn("forward short capped", "forward", 2, 8, 64, 512, cap=30.0),
        # Prefill of one long prompt, capped scores, wide heads: the largest.
        _attn("forward long capped", "forward", 1, 16, 128, 8192, cap=50.0),
        # Prefill of documents behind a bidirectional prefix, bias by buckets; an odd length.
        _attn("forward prefix buckets", "forward", 4, 12, 64, 2047, buckets=32, docs=True, prefix=True),
        # Training on packed documents with a linear distance bias.
        _attn("train linear bias docs", "train", 8, 12, 64, 2048, slopes=True, docs=True),
        # Training with capped scores, dense causal, wide heads.
        _attn("train capped dense", "train", 2, 16, 128, 2048, cap=50.0),
        # Training of a learned bias by distance buckets, one long document a row.
        _attn("train buckets", "train", 4, 16, 64, 2048, buckets=32),
        # Everything at once, an odd length, float16.
        _attn("train all ragged", "train", 3, 10, 128, 1531, cap=20.0, slopes=True, buckets=48, max_distance=400,
              docs=True, prefix=True, dtype="f16"),
        # Verification of sixteen drafts for each sequence of a full serving batch.
        _cache("tree batch 64", "tree", 64, 16, 64, 16, 512, 4096, 4096),
        # A large draft tree of one interactive sequence with a long cache, capped scores.
        _cache("tree single", "tree", 1, 16, 128, 61, 15000, 16384, 16384, cap=50.0),
        # One token of every sequence of a model with a linear distance bias and capped scores.
        _cache("token batch 64", "tree", 64, 16, 64, 1, 512, 4096, 4096, cap=30.0, slopes=True, chain=True),
        # Accepted drafts of a serving batch, and of one interactive sequence.
        _cache("commit batch 64", "commit", 64, 16, 64, 64, 16, 900, 1024, chain=True),
        _cache("commit single", "commit", 1, 12, 64, 5, 512, 1000, 1024),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["train", "train", "train", "forward", "forward", "tree", "tree", "tree", "commit"])
        head_dim = rng.choice([32, 64, 64, 64, 128, 128, 256])
        heads = max(2, _log_int(rng, 512, 2048) // head_dim)
        scores = {"cap": rng.choice([0.0, 15.0, 30.0, 50.0]), "slopes": rng.random() < 0.4,
                  "buckets": rng.choice([0, 0, 16, 32, 48, 64]), "max_distance": rng.choice([65, 128, 128, 256, 400, 512]),
                  "dtype": rng.choice(["bf16", "bf16", "bf16", "f16"])}
        if kind in ("tree", "commit"):
            storage = 8 * _log_int(rng, 64, 1024 if kind == "tree" else 128)
            lo = rng.randint(storage // 16, storage // 2)
            case = _cache("", kind, _log_int(rng, 1, 64), heads, head_dim, rng.choice([1, 1, _log_int(rng, 2, 64)]), lo,
                          rng.randint(lo, storage - 1), storage, ring=rng.choice([0, 0, 16, 64]),
                          chain=rng.random() < 0.3, **scores)
        else:
            case = _attn("", kind, _log_int(rng, 1, 16), heads, head_dim,
                         _log_int(rng, 100, 4096 if kind == "train" else 8192), docs=rng.random() < 0.6,
                         prefix=rng.random() < 0.3, **scores)
        del case["name"]
        w = work(case)
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES:
            return case


# Inputs -------------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _doc_lengths(case, seed):
    """Document lengths filling each row: log-normal around 400 tokens."""
    t, rows = case["tokens"], []
    g = torch.Generator().manual_seed(seed)
    for _ in range(case["batch"]):
        row, left = [], t
        while left:
            n = int(torch.empty(()).log_normal_(math.log(400.0), 0.8, generator=g).item())
            row.append(min(left, max(16, n)))
            left -= row[-1]
        rows.append(row)
    return rows


def _prefix_lengths(case, seed):
    g = torch.Generator().manual_seed(seed + 1)
    t = case["tokens"]
    return torch.randint(t // 8, t // 2 + 1, (case["batch"],), generator=g, dtype=torch.int32)


def _bucket_of(max_distance, buckets):
    """[max_distance + 1] int64: the bucket of each distance, the last entry also of every greater one. The first
    half of the buckets takes a distance each, the others grow geometrically; borders by whole numbers:
    e (M / e)^(j / m) <= n exactly where M^j e^m <= n^m e^j."""
    e = buckets // 2
    m = buckets - e
    out, j = [], 0
    for n in range(max_distance + 1):
        while n >= e and j + 1 < m and max_distance ** (j + 1) * e ** m <= n ** m * e ** (j + 1):
            j += 1
        out.append(n if n < e else e + j)
    return torch.tensor(out, device="cuda")


def _scores_state(case, g):
    """Slopes (a geometric sequence over the heads), the bias table and the buckets of the distances, as a model
    keeps them."""
    h, state = case["heads"], {"slopes": None, "table": None}
    if case["slopes"]:
        state["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda")
    if case["buckets"]:
        state["table"] = torch.randn((case["buckets"], h), generator=g, device="cuda").to(DTYPES[case["dtype"]])
        state["bucket"] = _bucket_of(case["max_distance"], case["buckets"])
    return state


def prepare(case, seed):
    return {"train": _prepare_attention, "forward": _prepare_attention, "tree": _prepare_cache,
            "commit": _prepare_cache}[case["kind"]](case, seed)


def _prepare_attention(case, seed):
    g, train = _gen(seed), case["kind"] == "train"
    b, h, n, d = case["batch"], case["heads"], case["tokens"], case["head_dim"]
    dtype = DTYPES[case["dtype"]]

    def rows(gain):
        x = torch.randn((b, n, h, d), generator=g, device="cuda") * gain
        return x.to(dtype).transpose(1, 2)

    state = {"case": case, **_scores_state(case, g), "qkv": [rows(GAIN), rows(GAIN), rows(1.0)], "docs": None,
             "prefix": None}
    if case["docs"]:
        ids = [torch.repeat_interleave(torch.arange(len(r)), torch.tensor(r)) for r in _doc_lengths(case, seed)]
        state["docs"] = torch.stack(ids).cuda()
    if case["prefix"]:
        state["prefix"] = _prefix_lengths(case, seed).cuda()
    if train:
        state["do"] = rows(1.0)
        state["leaves"] = [t.requires_grad_() for t in state["qkv"]]
        if state["table"] is not None:
            state["leaves"].append(state["table"].requires_grad_())
    return state


def _parents(case, seed):
    """Parents of the drafts of each sequence: a chain, or random trees of mostly recent parents."""
    b, t = case["batch"], case["drafts"]
    if case["chain"]:
        return torch.arange(-1, t - 1).repeat(b, 1).to(torch.int32)
    g = torch.Generator().manual_seed(seed + 2)
    i = torch.arange(t)[None]
    back = 1 + (torch.rand((b, t), generator=g) ** 2 * (i + 1)).long()
    return (i - back).clamp(min=-1).to(torch.int32)


def _prepare_cache(case, seed):
    g = _gen(seed)
    b, h, d, t, dtype = case["batch"], case["heads"], case["head_dim"], case["drafts"], DTYPES[case["dtype"]]

    def rand(*shape, gain=1.0):
        x = torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)
        return x.mul_(gain) if gain != 1.0 else x

    def lengths(lo, hi):
        return torch.randint(lo, hi + 1, (b,), generator=g, device="cuda")[:, None].expand(b, h).contiguous()

    state = {"case": case, **_scores_state(case, g), "q": rand(b, t, h, d, gain=GAIN),
             "draft_k": rand(b, t, h, d, gain=GAIN), "draft_v": rand(b, t, h, d),
             "parents": _parents(case, seed).cuda(),
             "k": [rand(b, h, case["storage"], d, gain=GAIN)], "v": [rand(b, h, case["storage"], d)],
             "len": [lengths(case["len_lo"], case["len_hi"])]}
    if case["ring"] and case["kind"] == "tree":
        state["k"].insert(0, rand(b, h, case["ring"], d, gain=GAIN))
        state["v"].insert(0, rand(b, h, case["ring"], d))
        state["len"].insert(0, torch.full((b,), case["ring"], dtype=torch.int64, device="cuda"))
    if case["kind"] == "commit":
        state["start"] = state["len"][0].clone()
        # The last accepted draft of each sequence, -1 where none was.
        state["last"] = torch.randint(-1, t, (b,), generator=g, device="cuda")
    return state


# One pass -----------------------------------------------------------------------------------------------


def run(state):
    if own:
        import sps_amd

        return {"forward": _own_forward, "train": _own_train, "tree": _own_tree,
                "commit": _own_commit}[state["case"]["kind"]](sps_amd, state)
    return {"forward": _plain_forward, "train": _plain_train, "tree": _plain_tree,
            "commit": _plain_commit}[state["case"]["kind"]](state)


def _changes(s):
    return {"softcap": s["case"]["cap"] or None, "slopes": s["slopes"], "bias_table": s["table"],
            "max_distance": s["case"]["max_distance"]}


def _own_attention(sps_amd, s):
    return sps_amd.biased_attention(*s["qkv"], s["case"]["head_dim"] ** -0.5, documents_idx_BxT=s["docs"],
                                    prefix_len_B=s["prefix"], **_changes(s))


def _own_forward(sps_amd, s):
    with torch.no_grad():
        return _own_attention(sps_amd, s)


def _own_train(sps_amd, s):
    o = _own_attention(sps_amd, s)
    return [o.detach(), *torch.autograd.grad(o, s["leaves"], s["do"])]


def _own_tree(sps_amd, s):
    segments = [sps_amd.KVSegment(k, v, n) for k, v, n in zip(s["k"], s["v"], s["len"])]
    return sps_amd.tree_attention(s["q"], segments, draft_k_BxTxHxD=s["draft_k"], draft_v_BxTxHxD=s["draft_v"],
                                  parents_BxT=None if s["case"]["chain"] else s["parents"], **_changes(s))


def _own_commit(sps_amd, s):
    s["len"][0].copy_(s["start"])  # every pass appends at the same lengths
    sps_amd.commit_drafts(sps_amd.KVSegment(s["k"][0], s["v"][0], s["len"][0]), s["draft_k"], s["draft_v"], s["last"],
                          parents_BxT=None if s["case"]["chain"] else s["parents"])
    return [s["k"][0], s["v"][0], s["len"][0]]


# Plain forms --------------------------------------------------------------------------------------------


def _plain_change(s, x, dist):
    """Scores x [H, ...] changed by cap and bias for distances `dist`, and the cap's derivative (None without)."""
    case, slope = s["case"], None
    if case["cap"]:
        t = torch.tanh(x / case["cap"])
        x, slope = t * case["cap"], 1 - t * t
    if s["slopes"] is not None:
        x = x - s["slopes"].reshape(-1, *[1] * (x.dim() - 1)) * dist.float()
    if s["table"] is not None:
        x = x + s["table"].detach().float().T[:, s["bucket"][dist.clamp(max=case["max_distance"])]]
    return x, slope


def _plain_softmax(x, hidden):
    """Softmax over the last axis of the scores that are not hidden; zeros where all are."""
    x = x.masked_fill(hidden, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, torch.ones_like(total), total)


def _plain_row(s, i, q, k):
    """Weights [H, N, N] of batch row i, the cap's derivative and the distances."""
    n = q.shape[1]
    at = torch.arange(n, device="cuda")
    see = at[None] <= at[:, None]
    if s["prefix"] is not None:
        see = see | (at[None] < s["prefix"][i])
    if s["docs"] is not None:
        see = see & (s["docs"][i][:, None] == s["docs"][i][None])
    dist = (at[:, None] - at[None]).clamp(min=0)
    x, slope = _plain_change(s, q @ k.transpose(1, 2) * s["case"]["head_dim"] ** -0.5, dist)
    return _plain_softmax(x, ~see), slope, dist


def _plain_forward(s):
    q, k, v = s["qkv"]
    rows = []
    for i in range(q.shape[0]):
        p, _, _ = _plain_row(s, i, q[i].float(), k[i].float())
        rows.append((p @ v[i].float()).to(q.dtype))
    return torch.stack(rows)


def _plain_table_gradient(s, ds):
    """Sums of ds [H, N, N] over the pairs of each bucket, [buckets, H]: by distance first. Row i of the flipped ds,
    moved i columns on, has the pairs of one distance in one column."""
    h, n, _ = ds.shape
    wide = torch.cat([ds.flip(2), torch.zeros_like(ds)], dim=2).reshape(h, 2 * n * n)[:, :n * (2 * n - 1)]
    sums = wide.reshape(h, n, 2 * n - 1).sum(1)
    by_dist, ahead = sums[:, n - 1:], sums[:, :n - 1].sum(1)
    bucket = s["bucket"][torch.arange(n, device="cuda").clamp(max=s["case"]["max_distance"])]
    one_hot = (bucket[:, None] == torch.arange(s["case"]["buckets"], device="cuda")).float()  # [N, buckets]
    total = (by_dist[:, :, None] * one_hot).sum(1)
    total[:, 0] += ahead
    return total.T


def _plain_train(s):
    case, dtype = s["case"], s["qkv"][0].dtype
    scale = case["head_dim"] ** -0.5
    outs, dq, dk, dv, dtable = [], [], [], [], 0.0
    for i in range(case["batch"]):
        q, k, v = (t.detach()[i].float() for t in s["qkv"])
        do = s["do"][i].float()
        p, slope, dist = _plain_row(s, i, q, k)
        o = p @ v
        dp = do @ v.transpose(1, 2)
        ds = p * (dp - (o * do).sum(-1, keepdim=True))
        if s["table"] is not None:
            dtable = dtable + _plain_table_gradient(s, ds)
        dx = ds if slope is None else ds * slope
        outs.append(o.to(dtype))
        dq.append((dx @ k * scale).to(dtype))
        dk.append((dx.transpose(1, 2) @ q * scale).to(dtype))
        dv.append((p.transpose(1, 2) @ do).to(dtype))
    outs = [torch.stack(x) for x in (outs, dq, dk, dv)]
    return outs + ([dtable.to(s["table"].dtype)] if s["table"] is not None else [])


def _ancestors(parents):
    """[B, T, T] bool: which drafts are a draft's ancestors or itself, and the drafts' depths [B, T]."""
    t = parents.shape[1]
    at = torch.arange(t, device="cuda")
    see = (at[:, None] == at) | (parents[..., None] == at)
    for _ in range((t - 1).bit_length()):  # steps of 1, 2, 4, ... generations
        see = (see.float() @ see.float()) > 0
    return see, see.sum(-1) - 1


def _plain_tree(s):
    case = s["case"]
    q = s["q"].float().transpose(1, 2)  # [B, H, T, D]
    b, h, t, d = q.shape
    see, depth = _ancestors(s["parents"])
    keys, values, shown, places, before = [], [], [], [], torch.zeros((b, h), dtype=torch.int64, device="cuda")
    for k, v, n in zip(s["k"], s["v"], s["len"]):
        n = n.reshape(b, -1).expand(b, h)
        at = torch.arange(k.shape[2], device="cuda")
        live = at < n[..., None]  # [B, H, S]
        keys.append(k.float())
        values.append(v.float())
        shown.append(live[:, :, None].expand(b, h, t, -1))
        places.append(before[..., None] + at)
        before = before + n
    keys.append(s["draft_k"].float().transpose(1, 2))
    values.append(s["draft_v"].float().transpose(1, 2))
    shown.append(see[:, None].expand(b, h, t, t))
    query_at = before[..., None] + depth[:, None]  # [B, H, T]
    places.append(query_at)
    key_at = torch.cat(places, dim=2)
    dist = (query_at[..., None] - key_at[:, :, None]).clamp(min=0)
    x = q @ torch.cat(keys, dim=2).transpose(2, 3) * d ** -0.5
    if case["cap"]:
        x = torch.tanh(x / case["cap"]) * case["cap"]
    if s["slopes"] is not None:
        x = x - s["slopes"][:, None, None] * dist.float()
    if s["table"] is not None:
        bucket = s["bucket"][dist.clamp(max=case["max_distance"])]
        x = x + s["table"].detach().float()[bucket, torch.arange(h, device="cuda")[:, None, None]]
    p = _plain_softmax(x, ~torch.cat(shown, dim=3))
    return (p @ torch.cat(values, dim=2)).transpose(1, 2).to(s["q"].dtype).contiguous()


def _plain_commit(s):
    lengths = s["len"][0]
    lengths.copy_(s["start"])
    see, depth = _ancestors(s["parents"])
    b, t = s["parents"].shape
    rows = torch.arange(b, device="cuda")
    last = s["last"]
    path = see[rows, last.clamp(min=0)] & (last >= 0)[:, None]  # [B, T]
    at = lengths[:, :, None] + depth[:, None]                   # [B, H, T]
    take = path[:, None] & (at < s["k"][0].shape[2])
    bi, hi, ti = take.nonzero(as_tuple=True)
    where = at[bi, hi, ti]
    s["k"][0][bi, hi, where] = s["draft_k"][bi, ti, hi]
    s["v"][0][bi, hi, where] = s["draft_v"][bi, ti, hi]
    lengths.add_(take.sum(-1))
    return [s["k"][0], s["v"][0], lengths]


# Work ---------------------------------------------------------------------------------------------------


def _pairs(case):
    """Visible (query, key) pairs of one head over the batch, for the documents and prefixes of seed 0."""
    total = 0
    prefixes = _prefix_lengths(case, 0).tolist() if case["prefix"] else [0] * case["batch"]
    lengths = _doc_lengths(case, 0) if case["docs"] else [[case["tokens"]]] * case["batch"]
    for row, prefix in zip(lengths, prefixes):
        first = 0
        for n in row:
            inside = min(max(prefix - first, 0), n)  # the document's part of the prefix: seen by its earlier queries too
            total += n * (n + 1) // 2 + inside * (inside - 1) // 2
            first += n
    return total


def work(case):
    h, d = case["heads"], case["head_dim"]
    if case["kind"] in ("forward", "train"):
        elems = case["batch"] * case["tokens"] * h * d
        train = case["kind"] == "train"
        return {"bytes": (8 if train else 4) * 2 * elems, "flops": (14.0 if train else 4.0) * _pairs(case) * h * d}
    rows, t = case["batch"] * h, case["drafts"]
    if case["kind"] == "tree":
        keys = (case["len_lo"] + case["len_hi"]) / 2 + case["ring"] + t
        return {"bytes": rows * (keys * d * 2 * 2 + 2 * t * d * 2), "flops": 4.0 * d * t * keys * rows}
    # Half the drafts of a chain lie on an accepted path, a few of a tree's; each row is read and written.
    taken = t / 2 if case["chain"] else min(t / 2, 4)
    return {"bytes": rows * (taken * d * 2 * 2 * 2 + 16), "flops": 0.0}


# 64-bit results -----------------------------------------------------------------------------------------


def exact(case, seed):
    if case["kind"] == "commit":
        return _exact_commit(case, seed)
    if case["kind"] == "tree":
        return _exact_tree(case, seed)
    return _exact_attention(case, seed)


def _exact_bias(s, n):
    """Bias of distances 0 .. n - 1 for each head, float64 [H, n]."""
    case = s["case"]
    dist = torch.arange(n, dtype=torch.float64, device="cuda")
    bias = torch.zeros((case["heads"], n), dtype=torch.float64, device="cuda")
    bucket = None
    if s["slopes"] is not None:
        bias = bias - torch.outer(s["slopes"].double(), dist)
    if s["table"] is not None:
        half = case["buckets"] // 2
        grown = (dist.clamp(min=half) / half).log() / math.log(case["max_distance"] / half) * (case["buckets"] - half)
        # Borders that are whole numbers come out a rounding below theirs.
        bucket = torch.where(dist < half, dist, half + (grown + 1e-9).floor()).clamp(max=case["buckets"] - 1).long()
        bias = bias + s["table"].detach().double()[bucket].T
    return bias, bucket


def _exact_scores(case, q, k, bias):
    """Changed scores and the cap's derivative of float64 queries and keys; `bias` matches the scores."""
    x = torch.einsum("qd,kd->qk", q, k) / math.sqrt(case["head_dim"])
    grow = 1.0
    if case["cap"]:
        c = torch.tanh(x / case["cap"])
        x, grow = case["cap"] * c, 1.0 - c.square()
    return x + bias, grow


def _exact_attention(case, seed):
    s = _prepare_attention(case, seed)
    b, h, n, d = case["batch"], case["heads"], case["tokens"], case["head_dim"]
    train = case["kind"] == "train"
    q, k, v = (t.detach() for t in s["qkv"])
    o = torch.empty((b, h, n, d), dtype=torch.float64, device="cuda")
    grads = [torch.empty_like(o) for _ in range(3)] if train else []
    dtable = torch.zeros((max(case["buckets"], 1), h), dtype=torch.float64, device="cuda")
    bias, bucket = _exact_bias(s, n)
    pos = torch.arange(n, device="cuda")
    dist = (pos.unsqueeze(1) - pos).relu()
    for i in range(b):
        hidden = pos.unsqueeze(1) < pos
        if s["prefix"] is not None:
            hidden &= pos >= s["prefix"][i]
        if s["docs"] is not None:
            hidden |= s["docs"][i].unsqueeze(1) != s["docs"][i]
        for j in range(h):
            qj, kj, vj = q[i, j].double(), k[i, j].double(), v[i, j].double()
            x, grow = _exact_scores(case, qj, kj, bias[j][dist])
            p = torch.softmax(x.masked_fill(hidden, -math.inf), dim=1)
            o[i, j] = p @ vj
            if not train:
                continue
            dj = s["do"][i, j].double()
            dp = dj @ vj.T
            ds = p * (dp - (p * dp).sum(1, keepdim=True))
            if bucket is not None:
                dtable[:, j].index_add_(0, bucket[dist].reshape(-1), ds.reshape(-1))
            dx = ds * grow / math.sqrt(d)
            for g, x in zip(grads, (dx @ kj, dx.T @ qj, p.T @ dj)):
                g[i, j] = x
    if not train:
        return o
    return [o, *grads] + ([dtable] if case["buckets"] else [])


def _exact_tree(case, seed):
    s = _prepare_cache(case, seed)
    b, h, t, d = case["batch"], case["heads"], case["drafts"], case["head_dim"]
    out = torch.empty((b, t, h, d), dtype=torch.float64, device="cuda")
    bias, _ = _exact_bias(s, sum(k.shape[2] for k in s["k"]) + t)
    parents = s["parents"].tolist()
    for i in range(b):
        lives = [int(n.reshape(b, -1)[i, 0]) for n in s["len"]]
        past = sum(lives)
        paths = []
        for x in range(t):
            p = parents[i][x]
            paths.append((paths[p] if p >= 0 else []) + [x])
        keys = torch.cat([k[i, :, :n] for k, n in zip(s["k"], lives)] + [s["draft_k"][i].transpose(0, 1)], dim=1).double()
        values = torch.cat([v[i, :, :n] for v, n in zip(s["v"], lives)] + [s["draft_v"][i].transpose(0, 1)], dim=1).double()
        depths = torch.tensor([len(p) - 1 for p in paths])
        places = torch.cat([torch.arange(past), past + depths]).cuda()
        hidden = torch.zeros((t, past + t), dtype=torch.bool)
        hidden[:, past:] = True
        for x, p in enumerate(paths):
            hidden[x, [past + y for y in p]] = False
        hidden = hidden.cuda()
        dist = (places[past:, None] - places).relu()
        for j in range(h):
            x, _ = _exact_scores(case, s["q"][i, :, j].double(), keys[j], bias[j][dist])
            out[i, :, j] = torch.softmax(x.masked_fill(hidden, -math.inf), dim=1) @ values[j]
    return out


def _exact_commit(case, seed):
    s = _prepare_cache(case, seed)
    k, v, lengths = s["k"][0], s["v"][0], s["start"].clone()
    parents, storage = s["parents"].tolist(), k.shape[2]
    for i, x in enumerate(s["last"].tolist()):
        path = []
        while x >= 0:
            path.insert(0, x)
            x = parents[i][x]
        n = int(lengths[i, 0])
        path = path[:storage - n]
        if path:
            k[i, :, n:n + len(path)] = s["draft_k"][i, path].transpose(0, 1)
            v[i, :, n:n + len(path)] = s["draft_v"][i, path].transpose(0, 1)
            lengths[i] += len(path)
    return [k.double(), v.double(), lengths]
