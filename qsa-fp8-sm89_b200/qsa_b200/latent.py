"""The latent cache: keys and values of all heads from one vector a token.

A token is ``rank`` latent values, which serve as key and value, and 64 rotated
ones, which serve as key. The paged cache keeps FP8 E4M3FN codes of the latent,
the rotated part in bf16 and one fp32 scale a token, a power of two::

    key = scale * (codes, rope)        value = scale * codes

Four calls serve one attention layer over it, asynchronous on the current CUDA
stream, CUDA tensors only:

* ``qsa_latent_append``: new latents (normed) and their rotated part into the
  cache;
* ``qsa_latent_decode``: the absorbed form, queries brought into the latent's
  space attend to the cache itself: whole contexts or Top-K selections, one
  token a request or a tree or chain of drafted ones;
* ``qsa_latent_read``: contexts out of the cache, to be expanded by the
  up-projection;
* ``qsa_latent_prefill``: the expanded form, for prompts.

The reference's caches hold a key and a value for each KV head
(sm89_cutedsl.py:48-62): ``qsa_decode`` serves those.
"""

from __future__ import annotations

import torch

from .block import _op


def latent_cache(num_pages: int, page_size: int, rank: int = 512, device="cuda"):
    """Empty cache ``(codes, rope, scales)``: E4M3FN ``[num_pages, page_size,
    rank]``, bf16 ``[num_pages, page_size, 64]``, fp32 ``[num_pages,
    page_size]``. ``rank`` is 128, 256, 384 or 512."""
    if rank not in (128, 256, 384, 512):
        raise ValueError(f"rank must be 128, 256, 384 or 512, got {rank}")
    codes = torch.zeros((num_pages, page_size, rank), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    rope = torch.zeros((num_pages, page_size, 64), dtype=torch.bfloat16, device=device)
    return codes, rope, torch.zeros((num_pages, page_size), device=device)


def qsa_latent_append(c_new, r_new, codes, rope, scales, btable, starts, *, reqs=None, cu_tokens=None, table=None,
                      positions=None, c_weight=None, eps=1e-6, interleaved=False):
    """Appends new tokens to the latent cache, in place.

    Entry e's tokens go to the logical positions ``starts[e]``, ``starts[e] +
    1``, ... of its request::

        y     = c * rsqrt(mean(c^2) + eps) * c_weight   (c itself without a weight)
        scale = 2^e, e the least with max|y| <= 448 * 2^e, from -60 to 60
        codes = e4m3fn(y / scale)                       ties to even, saturating
        rope  = bf16(rotated r / scale)

    Infinities of y count for no maximum and are stored as +-448; a token with
    a NaN in y gets the scale NaN (it reads as NaN) and zero codes. Tokens
    outside the block table or the cache are skipped.

    Args:
        c_new, r_new: bf16, fp16 or fp32 ``[tokens, rank]`` and ``[tokens,
            64]`` (views of a packed projection are taken).
        codes, rope, scales: see ``latent_cache``.
        btable: int32 ``[num_reqs, pages_per_req]``.
        starts: int32 ``[entries]``.
        reqs: int32 ``[entries]`` block-table rows (default: entry e's is e).
        cu_tokens: int32 ``[entries + 1]``, entry e has the tokens
            ``cu_tokens[e]`` to ``cu_tokens[e + 1] - 1``; None: one each.
        table: fp32 ``[positions, rotary_dim]`` (``rope_table``), rotary_dim a
            multiple of 16 up to 64; the rest passes through. None: no
            rotation.
        positions: int32 ``[tokens]`` for the rotation, such as the depths of
            drafted tokens; default: the logical positions. One outside the
            table gives a zero rotated part.
        c_weight: ``[rank]``, the latent's RMS norm; None: no norm.
        interleaved: pairs are neighbours (2j, 2j + 1); default (j, j +
            rotary_dim / 2).

    A place is named once in a call. Returns ``(codes, rope, scales)``.
    """
    _op("latent_append")(c_new, r_new, codes, rope, scales, btable, starts, reqs, cu_tokens, table, positions, c_weight,
                         eps, interleaved)
    return codes, rope, scales


def qsa_latent_read(codes, rope, scales, btable, starts, cu_tokens, tokens, *, reqs=None, dtype=torch.bfloat16, out=None):
    """Reads tokens back: ``scale * codes`` and ``scale * rope``, rounded once.

    Entry e's rows are the logical positions ``starts[e]``, ``starts[e] + 1``,
    ... of its request, laid out as in ``qsa_latent_append``; ``tokens`` is
    their number in all. Positions outside the block table or the cache give
    zeros, rows that no entry names are left as they are.

    Args:
        dtype: bf16, fp16 or fp32, of new outputs.
        out: optional pair of outputs, contiguous ``[tokens, rank]`` and
            ``[tokens, 64]`` of one such dtype.

    Returns ``(c, r)``.
    """
    if out is None:
        return _op("latent_read")(codes, rope, scales, btable, starts, cu_tokens, tokens, reqs, dtype)
    c, r = out
    if c.shape[0] != tokens:
        raise ValueError(f"the outputs have {c.shape[0]} rows, tokens is {tokens}")
    _op("latent_read_out")(codes, rope, scales, btable, starts, cu_tokens, reqs, c, r)
    return c, r


def qsa_latent_decode(q, codes, rope, scales, btable, t2r=None, indices=None, *, counts=None, tree=None, softmax_scale,
                      out=None):
    """Attention in the latent's space (the absorbed form)::

        out[r,i,h] = softmax_t(q[r,i,h] . key_t * softmax_scale) . value_t

    Args:
        q: bf16 ``[rows, heads, rank + 64]``, or ``[rows, nodes, heads, rank +
            64]`` for several query tokens of a row (contiguous, up to 128
            heads and 256 nodes): the queries through the keys' up-projection,
            then their rotated part.
        codes, rope, scales: see ``latent_cache``.
        btable: int32 ``[num_reqs, pages_per_req]``.
        t2r: int32 ``[rows]`` row -> block-table row, or None (identity).
        indices: int32 ``[rows, K]`` logical tokens (negative = masked), as
            ``qsa_topk_select`` gives them, with one node; None: every token
            in order.
        counts: int32 ``[rows]``: only the first ``counts[r]`` columns
            (without ``indices``: tokens) may be valid; default all.
        tree: int32 ``[rows, nodes, words]``. The row's nodes are the last
            ``nodes`` of its ``counts[r]`` tokens. Each sees the tokens before
            them and, of the nodes, those whose bit (j % 32 of word j // 32)
            is set; its own bit is an ancestor's like the others. None: a
            chain, node i sees nodes 0 to i. With one node it is not looked
            at: that node sees all its tokens.
        softmax_scale: as of the expanded form, such as ``192 ** -0.5``.
        out: optional bf16 output ``[rows, (nodes,) heads, rank]``.

    Masked entries (as in ``qsa_decode``) do not count; a node without a
    visible token gives zeros; a head whose query has an infinity or NaN gives
    NaN where it sees a token. Returns ``out``.
    """
    if out is None:
        return _op("latent_decode")(q, codes, rope, scales, btable, t2r, indices, counts, tree, softmax_scale)
    _op("latent_decode_out")(q, codes, rope, scales, btable, t2r, indices, counts, tree, softmax_scale, out)
    return out


def qsa_latent_prefill(q, k, k_rope, v, cu_q, cu_k=None, *, causal=True, softmax_scale=None, out=None):
    """Attention of prompts in the expanded form, over sequences of any
    lengths side by side::

        out[i,h] = softmax_j((q[i,h,:128] . k[j,h] + q[i,h,128:] . k_rope[j]) * softmax_scale) . v[j,h]

    Args:
        q: bf16 or fp16 ``[q_tokens, heads, 192]``.
        k, v: ``[k_tokens, heads, 128]``, such as views of one up-projection.
        k_rope: ``[k_tokens, 64]``, rotated, for all heads.
        cu_q: int32 ``[entries + 1]``: entry e has the query tokens
            ``cu_q[e]`` to ``cu_q[e + 1] - 1``.
        cu_k: the same for the key tokens; default ``cu_q``.
        causal: query i of an entry's n sees its keys up to i + (m - n) of m
            (a chunk behind cached tokens has m > n).
        softmax_scale: default ``192 ** -0.5``.
        out: optional output, contiguous ``[q_tokens, heads, 128]``.

    A query without a visible key gives zeros; query tokens that no entry
    names are left as they are. Returns ``out``.
    """
    if softmax_scale is None:
        softmax_scale = 192 ** -0.5
    if out is None:
        return _op("latent_prefill")(q, k, k_rope, v, cu_q, cu_k, causal, softmax_scale)
    _op("latent_prefill_out")(q, k, k_rope, v, cu_q, cu_k, causal, softmax_scale, out)
    return out
