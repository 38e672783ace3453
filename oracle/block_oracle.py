"""Block-scaled cache operators in 64 bits, from their definitions (numpy).

Test infrastructure: ``norm_rotate``, ``append`` and ``decode`` restate
``qsa_qk_rope``, ``qsa_block_append`` and ``qsa_block_decode``, each with the
size of the terms it sums, so that a test can derive its tolerance.
"""

from __future__ import annotations

import numpy as np

from .qsa_oracle import e4m3fn_table

D = 128
E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -126


def norm_rotate(x, weight=None, eps=1e-6, table=None, positions=None, sections=None, interleaved=False):
    """x [tokens, heads, 128] -> (y, size): the normed, rotated heads and, for
    each element, the sum of the absolute terms it is made of."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    y, size = x.copy(), np.abs(x)
    if table is None:
        return y, size
    table = np.asarray(table, np.float64)
    half = table.shape[1] // 2
    positions = np.asarray(positions)
    if positions.ndim == 1:
        positions = positions[None]
    ends = np.cumsum(sections) if sections is not None else [half]
    for j in range(half):
        axis = int(np.searchsorted(ends, j, side="right"))
        p = positions[axis]
        row = table[np.where((p >= 0) & (p < len(table)), p, 0)]
        c, s = row[:, j][:, None], row[:, half + j][:, None]
        i, k = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
        a, b = x[..., i], x[..., k]
        y[..., i], y[..., k] = a * c - b * s, b * c + a * s
        size[..., i] = np.abs(a * c) + np.abs(b * s)
        size[..., k] = np.abs(b * c) + np.abs(a * s)
    bad = ((positions < 0) | (positions >= len(table))).any(0)
    y[bad], size[bad] = 0.0, 0.0
    return y, size


def step(x):
    """Spacing of the E4M3FN values around |x|."""
    return np.exp2(np.floor(np.log2(np.clip(np.abs(x), 2.0 ** -6, E4M3_MAX))) - 3)


def append(k_new, v_new, k_cache, v_cache, k_scales, v_scales, btable, starts, reqs=None, cu_tokens=None):
    """Where and what ``qsa_block_append`` writes, keys given as normed and
    rotated. Caches are uint8 codes. Returns for K and for V a dict of
    ``scales`` (fp64, whole) and ``values`` (fp64 [pages, P, Hkv, 128]: code
    values before their rounding, NaN where the row stays as it was)."""
    n = len(starts)
    cu = np.arange(n + 1) if cu_tokens is None else np.asarray(cu_tokens)
    pages, page, hkv, _ = k_cache.shape
    block = page // k_scales.shape[1]
    tab = e4m3fn_table().astype(np.float64)
    out = []
    for x, cache, scales in ((k_new, k_cache, k_scales), (v_new, v_cache, v_scales)):
        x, new = np.asarray(x, np.float64), np.asarray(scales, np.float64).copy()
        values = np.full(cache.shape, np.nan)
        written = np.zeros(cache.shape[:2], bool)
        for e in range(n):
            req = e if reqs is None else int(reqs[e])
            if starts[e] < 0 or not 0 <= req < len(btable):
                continue
            start, count = int(starts[e]), int(cu[e + 1] - cu[e])
            if count == 0:
                continue
            for base in range(start - start % block, start + count, block):
                lp = base // page
                phys = int(btable[req][lp]) if lp < btable.shape[1] else -1
                if not 0 <= phys < pages:
                    continue
                off, b = base % page, base % page // block
                lo, hi = max(base, start), min(base + block, start + count)
                rows = x[cu[e] + lo - start:cu[e] + hi - start]
                finite = np.where(np.isfinite(rows), np.abs(rows), 0.0)
                old = np.asarray(scales, np.float64)[phys, b] if lo > base else np.zeros(hkv)
                s = np.maximum(old, np.maximum(finite.max((0, 2)) / E4M3_MAX, MIN_SCALE))
                new[phys, b] = s
                at = slice(off + lo - base, off + hi - base)
                values[phys, at] = rows / s[None, :, None]
                written[phys, at] = True
                kept = slice(off, off + lo - base)
                values[phys, kept] = tab[cache[phys, kept]] * (old / s)[None, :, None]
                written[phys, kept] = True
        out.append(dict(scales=new, values=values, written=written))
    return out


def decode(q, k_cache, v_cache, k_scales, v_scales, btable, t2r=None, indices=None, counts=None, gate=None,
           softmax_scale=None):
    """(out, size, score_size): the attention, for each output element the
    softmax average of |V|, and for each (row, head) the largest sum of
    absolute terms of a score."""
    q = np.asarray(q, np.float64)
    rows, hq, _ = q.shape
    pages, page, hkv, _ = k_cache.shape
    block = page // k_scales.shape[1]
    group = hq // hkv
    scale = D ** -0.5 if softmax_scale is None else softmax_scale
    tab = e4m3fn_table().astype(np.float64)
    out, size, ssize = np.zeros((rows, hq, D)), np.zeros((rows, hq, D)), np.zeros((rows, hq))
    for r in range(rows):
        req = r if t2r is None else int(t2r[r])
        if not 0 <= req < len(btable):
            continue
        cols = np.arange(btable.shape[1] * page) if indices is None else np.asarray(indices[r], np.int64)
        if counts is not None:
            cols = cols[:max(0, int(counts[r]))]
        cols = cols[(cols >= 0) & (cols // page < btable.shape[1])]
        phys = np.asarray(btable, np.int64)[req][cols // page]
        ok = (phys >= 0) & (phys < pages)
        cols, phys = cols[ok], phys[ok]
        if not len(cols):
            continue
        off = cols % page
        ks, vs = (np.asarray(s, np.float64)[phys, off // block] for s in (k_scales, v_scales))
        k, v = tab[k_cache[phys, off]] * ks[..., None], tab[v_cache[phys, off]] * vs[..., None]
        for h in range(hq):
            g = h // group
            score = k[:, g] @ q[r, h] * scale
            ssize[r, h] = (np.abs(k[:, g]) @ np.abs(q[r, h])).max() * abs(scale)
            p = np.exp(score - score.max())
            p /= p.sum()
            out[r, h], size[r, h] = p @ v[:, g], p @ np.abs(v[:, g])
    if gate is not None:
        s = 1 / (1 + np.exp(-np.asarray(gate, np.float64)))
        out, size = out * s, size * s
    return out, size, ssize
