"""Attention with changed scores in float64, forward and backward, with bounds of the kernels' rounding errors.

Test infrastructure only; the product never imports it. The definition is that of
sps_amd/biased_attention.py, written out densely.
"""

from __future__ import annotations

import numpy as np

HIDDEN = -16384.0  # table entries below hide their pairs


def bucket(n: int, num_buckets: int, max_distance: int) -> int:
    """Bucket of distance n, borders compared as whole numbers: (n / e)^m >= (M / e)^j."""
    e = num_buckets // 2
    m = num_buckets - e
    if n < e:
        return n
    j = 0
    while j + 1 < m and n ** m * e ** (j + 1) >= max_distance ** (j + 1) * e ** m:
        j += 1
    return e + j


def visible(n, docs=None, prefix=None):
    """[B, N, N] bool: k <= q or k < prefix[b], and equal document ids. docs [B, N], prefix [B]."""
    b = len(docs) if docs is not None else len(prefix) if prefix is not None else 1
    at = np.arange(n)
    see = np.broadcast_to(at[None, :] <= at[:, None], (b, n, n)).copy()
    if prefix is not None:
        see |= at[None, None, :] < np.asarray(prefix)[:, None, None]
    if docs is not None:
        d = np.asarray(docs)
        see &= d[:, :, None] == d[:, None, :]
    return see


def bias(h, n, slopes=None, table=None, max_distance=128):
    """[H, n] bias of distances 0 .. n - 1 (-inf where the table hides)."""
    out = np.zeros((h, n))
    if table is not None:
        t = np.where(np.asarray(table, np.float64) < HIDDEN, -np.inf, np.asarray(table, np.float64))
        out = out + t[[bucket(x, t.shape[0], max_distance) for x in range(n)]].T
    if slopes is not None:
        out = out - np.outer(np.asarray(slopes, np.float64), np.arange(n))
    return out


def weights(x, see):
    """Softmax over the last axis of the visible scores; zeros for rows with none."""
    x = np.where(see, x, -np.inf)
    top = x.max(-1, keepdims=True)
    with np.errstate(invalid="ignore"):
        p = np.where(np.isneginf(x), 0.0, np.exp(x - np.where(np.isfinite(top), top, 0.0)))
    total = p.sum(-1, keepdims=True)
    return p / np.where(total == 0, 1.0, total)


class Attention:
    """Dense forward and backward of [B, H, N, D] float64 arrays.

    Attributes after forward(): p, o; after backward(do): dq, dk, dv, dtable. ``bounds(dtype)`` gives, per result, how
    far the kernels' value may be from it: with u = eps / 2 of the inputs' type,
      - P and dS are rounded to that type for their products (u relative; float16 also 2^-25 absolute, its half step
        below 2^-14, against weights whose row maximum is at least 1);
      - weights, products and results below fp32's smallest normal value, 2^-126, may be flushed to zero;
      - Delta is summed from the rounded O, whose error is that of P's rounding and its own;
      - a score is off by its product's D fp32 additions, by the cap's difference (cap - 2 cap r, r within an ulp or
        two of the hardware's exponential and reciprocal) and by the roundings of the bias and log-sum-exp; a weight
        is off by that relative error, twice (numerator and normaliser);
      - each result is rounded once to its type.
    """

    def __init__(self, q, k, v, sm_scale, see, softcap=None, slopes=None, table=None, max_distance=128):
        self.q, self.k, self.v, self.scale, self.cap = q, k, v, float(sm_scale), softcap
        b, h, n, d = q.shape
        self.see = np.broadcast_to(see[:, None], (b, h, n, n))
        at = np.arange(n)
        self.dist = np.maximum(at[:, None] - at[None], 0)
        x = (q @ k.swapaxes(2, 3)) * self.scale
        self.slope = 1.0
        raw = (np.abs(q) @ np.abs(k).swapaxes(2, 3)) * abs(self.scale)
        if softcap:
            t = np.tanh(x / softcap)
            x, self.slope = softcap * t, 1.0 - t * t
        self.table, self.max_distance = table, max_distance
        bb = bias(h, n, slopes, table, max_distance)
        x = x + bb[:, self.dist][None]
        self.p = weights(x, self.see)
        self.o = self.p @ v
        e = 2.0 ** -24
        shown = self.see & np.isfinite(x)
        big = max([1.0, *np.abs(x[shown]).ravel()]) if shown.any() else 1.0
        slope_part = np.abs(np.asarray(slopes)).max() * n if slopes is not None else 0.0
        self.eps = 2 * ((d + 4) * e * (raw[shown].max() if shown.any() else 0.0) + 8 * e * (softcap or 0.0)
                        + 8 * e * (big + slope_part) + 16 * e)

    def backward(self, do):
        self.do = do
        self.dp = do @ self.v.swapaxes(2, 3)
        self.delta = (self.o * do).sum(-1, keepdims=True)
        self.ds = self.p * (self.dp - self.delta)
        dx = self.ds * self.slope * self.scale
        self.dq, self.dk, self.dv = dx @ self.k, dx.swapaxes(2, 3) @ self.q, self.p.swapaxes(2, 3) @ do
        self.dtable = None
        if self.table is not None:
            nb, h = self.table.shape
            buckets = np.array([bucket(x, nb, self.max_distance) for x in range(self.q.shape[2])])[self.dist]
            self.dtable = np.stack([[np.where(buckets == j, self.ds[:, i], 0.0).sum() for i in range(h)] for j in range(nb)])
            self._buckets = buckets

    def _units(self, dtype):
        return (2.0 ** -8, 2.0 ** -126) if dtype == "bf16" else (2.0 ** -11, 2.0 ** -25)

    def forward_bound(self, dtype):
        u, tiny = self._units(dtype)
        shown = self.see.astype(np.float64)
        return (u + self.eps) * (self.p @ np.abs(self.v)) + tiny * (shown @ np.abs(self.v)) + u * np.abs(self.o) + tiny

    def backward_bounds(self, dtype, table_unit=0.0):
        u, tiny = self._units(dtype)
        shown = self.see.astype(np.float64)
        d_o = self.forward_bound(dtype)
        d_delta = (np.abs(self.do) * d_o).sum(-1, keepdims=True) + 2.0 ** -20 * (np.abs(self.do) * np.abs(self.o)).sum(-1, keepdims=True)
        d_dp = 2.0 ** -18 * (np.abs(self.do) @ np.abs(self.v).swapaxes(2, 3))  # (256 fp32 additions)
        d_p = self.eps * self.p + 2.0 ** -126 * shown
        # dS before its rounding (what the table's gradient sums), and after it.
        d_ds = self.p * (d_delta + d_dp) + d_p * np.abs(self.dp - self.delta)
        scale = abs(self.scale)
        slope = np.abs(self.slope) * np.ones_like(self.p)
        d_dx = slope * (d_ds + u * np.abs(self.ds)) + u * d_ds + tiny * shown + 2.0 ** -20 * np.abs(self.ds)
        if self.cap:  # the derivative's own error, 4 r (1 - r) from r, and the raw score's
            d_dx = d_dx + np.abs(self.ds) * (self.eps + 2.0 ** -20)
        dq = scale * (d_dx @ np.abs(self.k)) + u * np.abs(self.dq) + tiny
        dk = scale * (d_dx.swapaxes(2, 3) @ np.abs(self.q)) + u * np.abs(self.dk) + tiny
        w = (u + self.eps) * self.p + tiny * shown
        dv = w.swapaxes(2, 3) @ np.abs(self.do) + u * np.abs(self.dv) + tiny
        out = [dq, dk, dv]
        if self.dtable is not None:
            nb, h = self.table.shape
            n = self.q.shape[2]
            e = d_ds + 2.0 ** -24 * (16 + n) * np.abs(self.ds)
            # A gradient in f16 below 2^-14, its least normal value, is rounded to a multiple of 2^-24: off by up to 2^-25,
            # whatever its size (1.474e-7 becomes 2 * 2^-24 = 1.192e-7). The other types' steps there are below 2^-126.
            least = 2.0 ** -25 if table_unit == 2.0 ** -11 else 2.0 ** -126
            out.append(np.stack([[np.where(self._buckets == j, e[:, i], 0.0).sum() for i in range(h)] for j in range(nb)])
                       + table_unit * np.abs(self.dtable) + least)
        return out


def finite_difference(f, x, i, step=1e-5):
    """Central difference of f along element i of array x (float64)."""
    y = x.copy()
    y[i] += step
    hi = f(y)
    y[i] -= 2 * step
    return (hi - f(y)) / (2 * step)


def tree_see(parents):
    """Ancestor-or-self matrix [T, T] and depths [T] (-1: no draft) of one sequence's parents: -1 a child of the cached
    tokens, an earlier draft its child, anything else (and whatever descends from it) no draft."""
    t = len(parents)
    see, depth = np.zeros((t, t), bool), np.full(t, -1)
    for i, p in enumerate(parents):
        if p == -1:
            depth[i] = 0
        elif 0 <= p < i and depth[p] >= 0:
            see[i] = see[p]
            depth[i] = depth[p] + 1
        else:
            continue
        see[i, i] = True
    return see, depth


def tree_attend(q, segments, draft_k, draft_v, parents, sm_scale, softcap=None, slopes=None, table=None,
                max_distance=128):
    """Tree attention in float64: q, draft_k, draft_v [B, T, H, D]; segments: (k, v [B, H, S, D], lengths [B] or
    [B, H], scan); parents [B, T]. Returns the outputs [B, T, H, D] and the weights' sums of |v| ([B, T, H, D])."""
    b, t, h, d = q.shape
    out, mag = np.zeros_like(q), np.zeros_like(q)
    for i in range(b):
        see, depth = tree_see(list(parents[i]))
        for j in range(h):
            keys, values = [], []
            for k, v, lengths, scan in segments:
                n = int(np.asarray(lengths)[i, j] if np.ndim(lengths) == 2 else lengths[i])
                n = max(0, min(n, k.shape[2], scan if scan is not None else k.shape[2]))
                keys.append(k[i, j, :n])
                values.append(v[i, j, :n])
            past = sum(len(x) for x in keys)
            own = depth >= 0
            keys, values = np.concatenate([*keys, draft_k[i, :, j]]), np.concatenate([*values, draft_v[i, :, j]])
            values = np.where(np.concatenate([np.ones(past, bool), own])[:, None], values, 0.0)
            keys = np.where(np.concatenate([np.ones(past, bool), own])[:, None], keys, 0.0)
            places = np.concatenate([np.arange(past), past + depth])
            dist = np.maximum((past + depth)[:, None] - places[None], 0)
            x = (q[i, :, j] @ keys.T) * sm_scale
            if softcap:
                x = softcap * np.tanh(x / softcap)
            one = lambda z: None if z is None else np.asarray(z)[..., j:j + 1]  # noqa: E731
            x = x + bias(1, past + t + 1, one(slopes), one(table), max_distance)[0][dist]
            shown = np.concatenate([np.broadcast_to(own[:, None], (t, past)), see], axis=1)
            p = weights(x, shown)
            out[i, :, j], mag[i, :, j] = p @ values, p @ np.abs(values)
    return out, mag


def tree_path(parents, last):
    """Drafts of the accepted path, root first; empty where `last` names no draft."""
    _, depth = tree_see(list(parents))
    if not 0 <= last < len(parents) or depth[last] < 0:
        return []
    path = []
    while last >= 0:
        path.insert(0, last)
        last = parents[last]
    return path


