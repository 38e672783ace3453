"""Latent cache operators in 64 bits, from their definitions (numpy).

Test infrastructure: ``append``, ``values``, ``decode`` and ``prefill`` restate
``qsa_latent_append``, ``qsa_latent_read``, ``qsa_latent_decode`` and
``qsa_latent_prefill``, with the sizes of the terms they sum, so that a test
can derive its tolerance.
"""

from __future__ import annotations

import numpy as np

from .qsa_oracle import e4m3fn_table

ROPE = 64
E4M3_MAX = 448.0
E_LOW, E_HIGH = -60, 60


def norm(c, weight=None, eps=1e-6):
    c = np.asarray(c, np.float64)
    if weight is None:
        return c
    return c / np.sqrt((c ** 2).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)


def rotate(r, table=None, positions=None, interleaved=False):
    """r [tokens, 64] -> (y, size): rotated, and the sum of absolute terms."""
    r = np.asarray(r, np.float64)
    y, size = r.copy(), np.abs(r)
    if table is None:
        return y, size
    table = np.asarray(table, np.float64)
    half = table.shape[1] // 2
    p = np.asarray(positions, np.int64)
    ok = (p >= 0) & (p < len(table))
    row = table[np.where(ok, p, 0)]
    for j in range(half):
        c, s = row[:, j], row[:, half + j]
        i, k = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
        a, b = r[:, i], r[:, k]
        y[:, i], y[:, k] = a * c - b * s, b * c + a * s
        size[:, i], size[:, k] = np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)
    y[~ok], size[~ok] = 0.0, 0.0
    return y, size


def exponent(top):
    """The least e with top <= 448 * 2^e, from -60 to 60."""
    mant, exp = np.frexp(np.asarray(top, np.float64))  # mant in [0.5, 1), 448 = 0.875 * 2^9
    e = exp - 9 + (mant > 0.875)
    return np.clip(np.where(np.asarray(top) > 0, e, E_LOW), E_LOW, E_HIGH)


def slots(btable, req, pos, page, pages):
    """Slots of a request's positions, -1 outside the table or the cache."""
    pos = np.asarray(pos, np.int64)
    lp = pos // page
    ok = (pos >= 0) & (lp < btable.shape[1])
    phys = np.asarray(btable, np.int64)[req][np.where(ok, lp, 0)]
    ok &= (phys >= 0) & (phys < pages)
    return np.where(ok, phys * page + pos % page, -1)


def places(btable, starts, reqs, cu_tokens, tokens, page, pages):
    """(named, position, slot) of every token of a call."""
    n = len(starts)
    cu = np.arange(n + 1) if cu_tokens is None else np.asarray(cu_tokens)
    named, pos, slot = np.zeros(tokens, bool), np.full(tokens, -1), np.full(tokens, -1)
    for e in range(n):
        req = e if reqs is None else int(reqs[e])
        a, b = int(cu[e]), int(cu[e + 1])
        named[a:b] = True
        if int(starts[e]) < 0 or not 0 <= req < len(btable):
            continue
        pos[a:b] = int(starts[e]) + np.arange(b - a)
        slot[a:b] = slots(btable, req, pos[a:b], page, pages)
    return named, pos, slot


def step(x):
    """Spacing of the E4M3FN values around |x|."""
    return np.exp2(np.floor(np.log2(np.clip(np.abs(x), 2.0 ** -6, E4M3_MAX))) - 3)


def values(codes, rope, scales):
    """Latent and rotated parts of a cache's tokens, flat: codes uint8, rope as
    numbers, scales as stored."""
    s = np.asarray(scales, np.float64).reshape(-1, 1)
    s = np.where(np.isnan(s), s, np.clip(s, 2.0 ** E_LOW, 2.0 ** E_HIGH))
    c = e4m3fn_table().astype(np.float64)[codes.reshape(-1, codes.shape[-1])]
    return c * s, np.asarray(rope, np.float64).reshape(-1, ROPE) * s


def visible(nodes, tree, columns, count):
    """Which columns (of `columns`, the first `count` valid) each node sees."""
    col = np.arange(columns)
    ok = np.repeat((col < count)[None], nodes, 0)
    if nodes > 1:
        for i in range(nodes):
            for j in range(nodes):
                at = count - nodes + j
                hidden = j > i if tree is None else not (int(tree[i, j // 32]) >> (j % 32)) & 1
                if hidden and 0 <= at < columns:
                    ok[i, at] = False
    return ok


def decode(q, codes, rope, scales, btable, t2r=None, indices=None, counts=None, tree=None, softmax_scale=1.0):
    """A list over rows of None (no visible token at all) or a dict: ``out``
    [nodes, heads, rank]; ``size``, the average of |value| by the same weights;
    ``score``, the largest sum of absolute terms of a score [nodes, heads];
    ``low``, the largest weight on the codes times the sum of |codes| over the
    columns [nodes, heads, rank]; ``low32``, the same of each 32 columns, summed
    over them; ``spread``, what independent relative errors of variance 1 of the
    weights give the average: the sum of (weight (value - out))^2; ``steps``, the
    same of errors of each 32 columns' largest weight on the codes."""
    rows, nodes, heads, _ = q.shape
    pages, page, rank = codes.shape
    lat, rot = values(codes, rope, scales)
    res = []
    for r in range(rows):
        req = r if t2r is None else int(t2r[r])
        cols = np.arange(btable.shape[1] * page) if indices is None else np.asarray(indices[r], np.int64)
        count = len(cols) if counts is None else max(0, int(counts[r]))
        if not 0 <= req < len(btable):
            res.append(None)
            continue
        ok = visible(nodes, None if tree is None else tree[r], len(cols), count)
        at = slots(btable, req, cols, page, pages)
        ok &= (at >= 0)[None]
        any_col = ok.any(0)
        if not any_col.any():
            res.append(None)
            continue
        at, ok = at[any_col], ok[:, any_col]
        c, x = lat[at], rot[at]
        key = np.concatenate([c, x], 1)
        s = np.abs(np.asarray(scales, np.float64).reshape(-1)[at])
        with np.errstate(invalid="ignore"):
            score = np.einsum("nhd,td->nht", np.asarray(q[r], np.float64), key) * softmax_scale
            terms = np.einsum("nhd,td->nht", np.abs(np.asarray(q[r], np.float64)), np.abs(key)) * abs(softmax_scale)
        score = np.where(ok[:, None], score, -np.inf)
        seen = ok.any(1)
        top = np.where(seen[:, None], score.max(-1), 0.0)
        with np.errstate(invalid="ignore"):
            p = np.where(ok[:, None], np.exp(score - top[..., None]), 0.0)
        p = p / np.where(seen[:, None], p.sum(-1), 1.0)[..., None]
        c0 = np.where(np.isnan(c), 0.0, c)  # a token that a node does not see has no part in it

        def mix(w, x):
            out = np.einsum("nht,td->nhd", np.where(np.isnan(w), 0.0, w), x)
            out[np.isnan(w).any(-1)] = np.nan
            return out

        codes_abs = np.abs(c0) / np.where(s > 0, s, 1.0)[:, None]
        with np.errstate(invalid="ignore"):
            on_codes = np.where((p > 0) & np.isfinite(s), p * s, 0.0)  # of a head with a NaN weight nothing is compared
        low = on_codes.max(-1)[..., None] * codes_abs.sum(0)
        cuts = np.flatnonzero(np.diff(np.flatnonzero(any_col) // 32, prepend=-1))  # where another 32 columns begin
        largest = np.maximum.reduceat(on_codes, cuts, axis=-1)
        low32 = np.einsum("nhb,bd->nhd", largest, np.add.reduceat(codes_abs, cuts, axis=0))
        steps = np.einsum("nhb,bd->nhd", largest ** 2, np.add.reduceat(codes_abs ** 2, cuts, axis=0))
        out, p0 = mix(p, c0), np.where(np.isnan(p), 0.0, p) ** 2
        spread = np.einsum("nht,td->nhd", p0, c0 ** 2) - 2 * out * np.einsum("nht,td->nhd", p0, c0) + out ** 2 * p0.sum(-1)[..., None]
        res.append(dict(out=out, size=mix(p, np.abs(c0)), score=np.where(ok[:, None], terms, 0.0).max(-1), low=low, low32=low32,
                        spread=spread, steps=steps))
    return res


def prefill(q, k, k_rope, v, cu_q, cu_k, causal, softmax_scale):
    """(out, size, score, named) of the expanded form: the softmax average of
    |v|, and the largest sum of absolute terms of a score."""
    tokens, heads = q.shape[:2]
    out, size, score_size = np.zeros((tokens, heads, 128)), np.zeros((tokens, heads, 128)), np.zeros((tokens, heads))
    named = np.zeros(tokens, bool)
    for e in range(len(cu_q) - 1):
        a, b, c, d = int(cu_q[e]), int(cu_q[e + 1]), int(cu_k[e]), int(cu_k[e + 1])
        named[a:b] = True
        if a == b or c == d:
            continue
        for h in range(heads):
            key = np.concatenate([k[c:d, h], k_rope[c:d]], 1)
            score = q[a:b, h] @ key.T * softmax_scale
            terms = np.abs(q[a:b, h]) @ np.abs(key).T * abs(softmax_scale)
            ok = np.ones(score.shape, bool)
            if causal:
                ok = np.arange(d - c)[None] <= np.arange(b - a)[:, None] + (d - c) - (b - a)
            score = np.where(ok, score, -np.inf)
            seen = ok.any(1)
            p = np.exp(score - np.where(seen, score.max(1), 0.0)[:, None])
            p /= np.where(seen, p.sum(1), 1.0)[:, None]
            out[a:b, h], size[a:b, h] = p @ v[c:d, h], p @ np.abs(v[c:d, h])
            score_size[a:b, h] = np.where(ok, terms, 0.0).max(1)
    return out, size, score_size, named
