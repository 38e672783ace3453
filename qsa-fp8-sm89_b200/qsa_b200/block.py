"""The block-scaled paged cache: FP8 E4M3FN codes with one fp32 scale for each
block of consecutive tokens and KV head.

    stored value = code * scales[page, (t % P) // block, g]

Three calls serve one attention layer over it, asynchronous on the current
CUDA stream, CUDA tensors only. Each is one launch; the decode of rows of more
than 512 columns is three, or four with ``indices``:

* ``qsa_qk_rope``: RMS norm of every query and key head and the position
  rotation, over one or several position axes, in one pass;
* ``qsa_block_append``: new keys (normed and rotated on the way) and values
  into the cache, with the scales of the blocks they fall in;
* ``qsa_block_decode``: attention over Top-K selections or whole contexts.

The reference's caches have one scale each (sm89_cutedsl.py:48-62, :79) and
hold what they are given: ``qsa_cache_write`` and ``qsa_decode`` serve those.
"""

from __future__ import annotations

import torch

from ._lib import load_torch_ops

_ops: dict = {}


def _op(name: str):
    """The registered overload, looked up once."""
    op = _ops.get(name)
    if op is None:
        op = _ops[name] = getattr(load_torch_ops(), name).default
    return op


def rope_table(length: int, rotary_dim: int = 128, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """Rotation table, fp32 ``[length, rotary_dim]``: the cosines, then the
    sines, of position * theta^(-2j / rotary_dim), computed in 64 bits (an
    fp32 angle would be off by 2^-24 of itself, 0.06 rad at position 2^20)."""
    freq = float(theta) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], dim=1).to(torch.float32)


def block_cache(num_pages: int, page_size: int, num_kv_heads: int, block_size: int | None = None, device="cuda"):
    """Empty caches and scales ``(k_cache, v_cache, k_scales, v_scales)``:
    E4M3FN ``[num_pages, page_size, num_kv_heads, 128]`` and fp32 ``[num_pages,
    page_size // block_size, num_kv_heads]`` (default: one block a page)."""
    block = page_size if block_size is None else int(block_size)
    if block < 1 or page_size % block:
        raise ValueError(f"block_size must divide the page of {page_size} tokens, got {block_size}")
    shape = (num_pages, page_size, num_kv_heads, 128)
    caches = [torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.zeros((num_pages, page_size // block, num_kv_heads), device=device) for _ in range(2)]
    return (*caches, *scales)


def qsa_qk_rope(q, k=None, table=None, positions=None, *, q_weight=None, k_weight=None, eps=1e-6, interleaved=False,
                sections=None, q_out=None, k_out=None):
    """RMS norm of every query and key head and the position rotation::

        y = x * rsqrt(mean(x^2) + eps) * weight, then rotated

    in fp32, rounded once to the inputs' dtype.

    Args:
        q, k: bf16, fp16 or fp32 ``[tokens, heads, 128]``, heads contiguous
            (views of a packed projection are taken); ``k`` may be None.
        table: fp32 ``[positions, rotary_dim]`` cosines, then sines
            (``rope_table``), rotary_dim a multiple of 16 up to 128; the rest
            of the head passes through. None: no rotation.
        positions: int32 ``[tokens]``, or ``[axes, tokens]`` with
            ``sections``. A token with a position outside the table gives
            zeros.
        q_weight, k_weight: ``[128]``, one dtype of the three; None: no norm.
        interleaved: pairs are neighbours (2j, 2j + 1); default (j, j +
            rotary_dim / 2).
        sections: pairs of each axis, such as (16, 24, 24) for time, height
            and width; they sum to rotary_dim / 2.
        q_out, k_out: outputs, new by default; the inputs themselves rotate in
            place.

    Returns ``(q_out, k_out)``, ``k_out`` None without ``k``.
    """
    if q_out is None and k_out is None:
        q_out, k_out = _op("qk_rope")(q, k, table, positions, q_weight, k_weight, eps, interleaved, sections)
        return q_out, k_out if k is not None else None
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if k is not None and k_out is None:
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    _op("qk_rope_out")(q, k, table, positions, q_weight, k_weight, eps, interleaved, sections, q_out, k_out)
    return q_out, k_out


def qsa_block_append(k_new, v_new, k_cache, v_cache, k_scales, v_scales, btable, starts, *, reqs=None, cu_tokens=None,
                     table=None, positions=None, k_weight=None, eps=1e-6, interleaved=False, sections=None):
    """Appends new keys and values to the block-scaled caches, in place.

    Entry e's tokens go to the logical positions ``starts[e]``, ``starts[e] +
    1``, ... of its request. For each block and head that gets a token::

        s = max(s_old, max|x| / 448, 2^-126)     over the block's new rows x
        new rows  = e4m3fn(x / s)                ties to even, saturating
        kept rows = e4m3fn(code * (s_old / s))

    with ``s_old`` the block's scale where it keeps tokens before
    ``starts[e]``, else 0: a page that comes back from another request needs
    no clearing. Infinities count for no maximum and are stored as +-448, NaN
    stays NaN. Tokens outside the block table or the cache are skipped.

    Args:
        k_new, v_new: bf16, fp16 or fp32 ``[tokens, Hkv, 128]``, heads
            contiguous, one token stride for both.
        k_cache, v_cache, k_scales, v_scales: see ``block_cache``.
        btable: int32 ``[num_reqs, pages_per_req]``.
        starts: int32 ``[entries]``.
        reqs: int32 ``[entries]`` block-table rows (default: entry e's is e).
        cu_tokens: int32 ``[entries + 1]``, entry e has the tokens
            ``cu_tokens[e]`` to ``cu_tokens[e + 1] - 1``; None: one each.
        table, positions, interleaved, sections: the keys' rotation, as in
            ``qsa_qk_rope``; without ``positions`` by the logical positions.
        k_weight, eps: the keys' norm, as in ``qsa_qk_rope``.

    A page that gets tokens belongs to one request, and a request comes once
    in a call. Returns ``(k_cache, v_cache, k_scales, v_scales)``.
    """
    _op("block_append")(k_new, v_new, k_cache, v_cache, k_scales, v_scales, btable, starts, reqs, cu_tokens, table,
                        positions, k_weight, eps, interleaved, sections)
    return k_cache, v_cache, k_scales, v_scales


def qsa_block_decode(q, k_cache, v_cache, k_scales, v_scales, btable, t2r, indices=None, *, gate=None, counts=None,
                     softmax_scale=None, out=None):
    """Grouped-query attention over the block-scaled caches::

        out[r,h] = softmax_t(q[r,h] . K[t,g] ks[t,g] softmax_scale) . V[t,g] vs[t,g]
                   * sigmoid(gate[r,h])

    Args:
        q: bf16 ``[rows, Hq, 128]`` (contiguous), Hq / Hkv from 1 to 32.
        k_cache, v_cache, k_scales, v_scales: see ``block_cache``.
        btable: int32 ``[num_reqs, pages_per_req]``.
        t2r: int32 ``[rows]`` row -> block-table row, or None (identity).
        indices: int32 ``[rows, K]`` logical tokens (negative = masked), as
            ``qsa_topk_select`` gives them; None: every token in order.
        gate: optional bf16 like ``q``.
        counts: optional int32 ``[rows]``: only the first ``counts[r]``
            columns (without ``indices``: tokens) may be valid.
        softmax_scale: default ``D ** -0.5``.
        out: optional bf16 output like ``q``.

    Masked entries (as in ``qsa_decode``) are not read; a row without a valid
    entry gives zeros. Returns ``out``.
    """
    if softmax_scale is None:
        softmax_scale = q.shape[-1] ** -0.5
    if out is None:
        return _op("block_decode")(q, k_cache, v_cache, k_scales, v_scales, btable, t2r, indices, gate, counts,
                                   softmax_scale)
    _op("block_decode_out")(q, k_cache, v_cache, k_scales, v_scales, btable, t2r, indices, gate, counts, softmax_scale,
                            out)
    return out
