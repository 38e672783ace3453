"""The block-scaled cache: qsa_qk_rope, qsa_block_append, qsa_block_decode.

CPU: the 64-bit oracle against hand-made values, and the C ABI's refusals
(they run before any device is touched). GPU: each operator against the oracle
at the sizes, masks and values where it can go wrong.

Tolerances, with u = 2^-24 the fp32 rounding:

* qk_rope: an element is a norm (12 roundings of the sum of squares, halved by
  the root, 2 ulp of rsqrtf, 3 products) and two rotation products and a sum:
  under 16 u of its terms' size; then one rounding to the output's type.
* append: the scale carries a key's 16 u and one division's; a code is the
  nearest to x / s, off by half a step, the key's error and 4 u of x / s.
* decode: scores accumulate 128 products in fp32 (under 2^-17 of the size of
  their terms, which moves a probability by as much); probabilities and the
  scale they carry may be rounded to 11 bits (2^-11 each way); 2^-12 for the
  sums; then one bf16 rounding (8 significant bits: 2^-8).
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import block_oracle as B
from oracle import qsa_oracle as O

D = 128
U = 2.0 ** -24
ROUND = {torch.float32: (0.0, 0.0), torch.float16: (2.0 ** -11, 2.0 ** -25), torch.bfloat16: (2.0 ** -8, 2.0 ** -133)}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def np64(t):
    return t.detach().double().cpu().numpy()


def u8(t):
    return t.detach().view(torch.uint8).cpu().numpy()


def rope_table(n, rotary):
    from qsa_b200 import rope_table as table

    return table(n, rotary, 10000.0, device="cpu")


# ------------------------------------------------------------------- CPU ----
def test_rope_table_is_rounded_from_64_bits():
    t = rope_table(70001, 32)
    ang = 70000 * 10000.0 ** (-np.arange(16) / 16)
    assert t.shape == (70001, 32) and t.dtype == torch.float32
    assert np.array_equal(t[70000].numpy(), np.concatenate([np.cos(ang), np.sin(ang)]).astype(np.float32))


def test_oracle_rotation_turns_pairs():
    x = np.zeros((1, 1, D))
    x[0, 0, 1], x[0, 0, 9] = 3.0, 4.0
    table = np.zeros((2, 16))
    table[:, :8], table[1, 1], table[1, 9] = 1.0, 0.0, 1.0  # position 1 turns pair 1 by 90 degrees
    y, _ = B.norm_rotate(x, table=table, positions=[1])
    assert y[0, 0, 1] == -4.0 and y[0, 0, 9] == 3.0  # halves: (1, 9)
    y, _ = B.norm_rotate(x, table=table, positions=[1], interleaved=True)
    assert y[0, 0, 1] == 3.0 and y[0, 0, 9] == 4.0  # pair 1 is (2, 3)
    y, _ = B.norm_rotate(x, table=table, positions=[[0], [1]], sections=(1, 7))
    assert y[0, 0, 1] == -4.0  # pair 1 goes by the second axis
    assert not B.norm_rotate(x, table=table, positions=[2])[0].any()


def test_oracle_append_grows_a_kept_block_and_restarts_a_fresh_one():
    kc = np.full((2, 4, 1, D), 0x38, np.uint8)  # code 1.0
    ks = np.full((2, 2, 1), 1.0 / 448)
    x = np.full((2, 1, D), 2.0)
    k, _ = B.append(x, x, kc, kc, ks, ks, np.array([[0, 1]]), [1], cu_tokens=[0, 2])
    # positions 1 and 2: block 0 keeps token 0 and grows to 2 / 448, block 1 starts anew
    assert np.allclose(k["scales"][0, :, 0], [2 / 448, 2 / 448])
    assert np.allclose(k["values"][0, 0], 0.5) and np.allclose(k["values"][0, 1:3], 448.0)
    assert np.isnan(k["values"][0, 3]).all() and np.isnan(k["values"][1]).all()


def _rope_args(**over):
    from qsa_b200 import capi

    a = capi.QkRopeArgs()
    a.q, a.k, a.q_out, a.k_out, a.q_weight, a.k_weight = (ctypes.c_void_p(0x10000 * (i + 1)) for i in range(6))
    a.eps, a.tokens, a.num_q_heads, a.num_kv_heads, a.head_dim = 1e-6, 4, 8, 2, 128
    a.q_stride = a.q_out_stride = 1024
    a.k_stride = a.k_out_stride = 256
    a.rope = _rotation()
    for k, v in over.items():
        setattr(a.rope if hasattr(a.rope, k) else a, k, v)
    return a


def _rotation():
    from qsa_b200 import capi

    r = capi.Rotation()
    r.table, r.positions = ctypes.c_void_p(0x100000), ctypes.c_void_p(0x110000)
    r.table_len, r.rotary_dim, r.num_axes, r.axis_stride = 100, 128, 1, 4
    return r


def _sections(*s):
    from qsa_b200 import capi

    return (ctypes.c_int32 * capi.ROPE_MAX_AXES)(*s)


def test_qk_rope_refuses_bad_arguments_before_the_device():
    from qsa_b200 import capi

    assert capi.lib().qsa_b200_qk_rope(None, None) == capi.ERR_NULL_POINTER
    for over, want in [
        (dict(head_dim=64), capi.ERR_UNSUPPORTED),
        (dict(dtype=3), capi.ERR_UNSUPPORTED),
        (dict(weight_dtype=-1), capi.ERR_UNSUPPORTED),
        (dict(eps=float("nan")), capi.ERR_BAD_VALUE),
        (dict(eps=-1e-6), capi.ERR_BAD_VALUE),
        (dict(tokens=-1), capi.ERR_BAD_SHAPE),
        (dict(num_q_heads=0), capi.ERR_BAD_SHAPE),
        (dict(num_kv_heads=0), capi.ERR_BAD_SHAPE),
        (dict(q_stride=1023), capi.ERR_BAD_SHAPE),
        (dict(k_out_stride=255), capi.ERR_BAD_SHAPE),
        (dict(q=None), capi.ERR_NULL_POINTER),
        (dict(k_out=None), capi.ERR_NULL_POINTER),
        (dict(positions=None), capi.ERR_NULL_POINTER),
        (dict(rotary_dim=24), capi.ERR_UNSUPPORTED),
        (dict(rotary_dim=144), capi.ERR_UNSUPPORTED),
        (dict(num_axes=5), capi.ERR_UNSUPPORTED),
        (dict(num_axes=2, sections=_sections(32, 31)), capi.ERR_BAD_SHAPE),
        (dict(num_axes=2, sections=_sections(-1, 65)), capi.ERR_BAD_SHAPE),
        (dict(num_axes=2, sections=_sections(32, 32), axis_stride=3), capi.ERR_BAD_SHAPE),
        (dict(table_len=0), capi.ERR_BAD_SHAPE),
        (dict(q=ctypes.c_void_p(0x10008)), capi.ERR_MISALIGNED),
        (dict(q_stride=1028), capi.ERR_MISALIGNED),
        (dict(k_weight=ctypes.c_void_p(0x60004)), capi.ERR_MISALIGNED),
        (dict(table=ctypes.c_void_p(0x100004)), capi.ERR_MISALIGNED),
        (dict(positions=ctypes.c_void_p(0x110002)), capi.ERR_MISALIGNED),
    ]:
        assert capi.qk_rope(_rope_args(**over)) == want, over
    assert capi.qk_rope(_rope_args(tokens=0)) == capi.OK


def _append_args(**over):
    from qsa_b200 import capi

    a = capi.BlockAppendArgs()
    for i, f in enumerate(("k", "v", "k_cache", "v_cache", "k_scales", "v_scales", "btable", "starts", "cu_tokens")):
        setattr(a, f, ctypes.c_void_p(0x10000 * (i + 1)))
    a.eps, a.entries, a.tokens, a.num_kv_heads, a.head_dim = 1e-6, 3, 10, 8, 128
    a.page_size, a.block_size, a.pages_per_req, a.num_reqs, a.num_pages = 16, 8, 4, 3, 64
    a.btable_stride, a.token_stride = 4, 1024
    a.rope = _rotation()
    a.rope.axis_stride = 10
    for k, v in over.items():
        setattr(a.rope if hasattr(a.rope, k) else a, k, v)
    return a


def test_block_append_refuses_bad_arguments_before_the_device():
    from qsa_b200 import capi

    assert capi.lib().qsa_b200_block_append(None, None) == capi.ERR_NULL_POINTER
    for over, want in [
        (dict(block_size=6), capi.ERR_BAD_SHAPE),
        (dict(block_size=0), capi.ERR_BAD_SHAPE),
        (dict(page_size=0), capi.ERR_BAD_SHAPE),
        (dict(btable_stride=3), capi.ERR_BAD_SHAPE),
        (dict(num_pages=0), capi.ERR_BAD_SHAPE),
        (dict(entries=-1), capi.ERR_BAD_SHAPE),
        (dict(cu_tokens=None), capi.ERR_BAD_SHAPE),  # 10 tokens, 3 entries
        (dict(token_stride=1023), capi.ERR_BAD_SHAPE),
        (dict(head_dim=256), capi.ERR_UNSUPPORTED),
        (dict(input_dtype=9), capi.ERR_UNSUPPORTED),
        (dict(rotary_dim=8), capi.ERR_UNSUPPORTED),
        (dict(num_axes=2, positions=None, sections=_sections(32, 32)), capi.ERR_NULL_POINTER),
        (dict(eps=float("inf")), capi.ERR_BAD_VALUE),
        (dict(starts=None), capi.ERR_NULL_POINTER),
        (dict(v_scales=None), capi.ERR_NULL_POINTER),
        (dict(v=ctypes.c_void_p(0x20008)), capi.ERR_MISALIGNED),
        (dict(token_stride=1028), capi.ERR_MISALIGNED),
        (dict(k_scales=ctypes.c_void_p(0x50002)), capi.ERR_MISALIGNED),
    ]:
        assert capi.block_append(_append_args(**over)) == want, over
    for over in (dict(tokens=0), dict(entries=0)):
        assert capi.block_append(_append_args(**over)) == capi.OK


def _decode_args(**over):
    from qsa_b200 import capi

    a = capi.BlockDecodeArgs()
    for i, f in enumerate(("q", "k_cache", "v_cache", "k_scales", "v_scales", "indices", "btable", "gate", "out")):
        setattr(a, f, ctypes.c_void_p(0x10000 * (i + 1)))
    a.softmax_scale, a.rows, a.num_q_heads, a.num_kv_heads, a.head_dim = 0.1, 4, 32, 8, 128
    a.page_size, a.block_size, a.pages_per_req, a.num_reqs, a.num_pages = 16, 16, 8, 4, 64
    a.topk, a.indices_stride, a.btable_stride = 100, 100, 8
    for k, v in over.items():
        setattr(a, k, v)
    return a


def test_block_decode_refuses_bad_arguments_before_the_device():
    from qsa_b200 import capi

    assert capi.lib().qsa_b200_block_decode(None, None, 0, None) == capi.ERR_NULL_POINTER
    assert capi.lib().qsa_b200_block_decode_workspace_bytes(None) == capi.ERR_NULL_POINTER
    for over, want in [
        (dict(head_dim=64), capi.ERR_UNSUPPORTED),
        (dict(num_q_heads=33 * 8), capi.ERR_UNSUPPORTED),
        (dict(num_pages=1 << 27), capi.ERR_UNSUPPORTED),  # 2^31 slots
        (dict(indices=None, pages_per_req=1 << 27, btable_stride=1 << 27), capi.ERR_UNSUPPORTED),
        (dict(num_q_heads=30), capi.ERR_BAD_SHAPE),
        (dict(rows=-1), capi.ERR_BAD_SHAPE),
        (dict(block_size=5), capi.ERR_BAD_SHAPE),
        (dict(topk=-1), capi.ERR_BAD_SHAPE),
        (dict(indices_stride=99), capi.ERR_BAD_SHAPE),
        (dict(btable_stride=7), capi.ERR_BAD_SHAPE),
        (dict(k_scales=None), capi.ERR_NULL_POINTER),
        (dict(out=None), capi.ERR_NULL_POINTER),
        (dict(q=ctypes.c_void_p(0x10008)), capi.ERR_MISALIGNED),
        (dict(gate=ctypes.c_void_p(0x80002)), capi.ERR_MISALIGNED),
        (dict(v_scales=ctypes.c_void_p(0x50001)), capi.ERR_MISALIGNED),
    ]:
        assert capi.block_decode(_decode_args(**over)) == want, over
        assert capi.block_decode_workspace_bytes(_decode_args(**over)) == want, over
    assert capi.block_decode(_decode_args(rows=0)) == capi.OK
    assert capi.block_decode_workspace_bytes(_decode_args(rows=0)) == 0


def test_block_cache_refuses_an_uneven_block():
    from qsa_b200 import block_cache

    with pytest.raises(ValueError):
        block_cache(4, 16, 2, 5, device="cpu")
    k, v, ks, vs = block_cache(4, 16, 2, 8, device="cpu")
    assert k.shape == v.shape == (4, 16, 2, 128) and ks.shape == vs.shape == (4, 2, 2)


# --------------------------------------------------------------- GPU: rope ----
ROPE_CASES = [
    # tokens, hq, hkv, rotary, interleaved, sections, norm
    (1, 1, 1, 128, False, None, True),
    (1, 32, 8, 128, False, None, True),
    (3, 5, 2, 16, False, None, True),
    (7, 3, 0, 48, False, None, False),
    (5, 8, 1, 112, True, None, True),
    (33, 24, 4, 128, False, (16, 24, 24), True),
    (18, 6, 3, 64, True, (5, 11, 16), True),
    (9, 2, 2, 32, False, (0, 3, 13, 0), False),
    (4, 4, 1, 0, False, None, True),
    (700, 64, 8, 128, False, None, True),
]


def _rope_check(got, x, weight, table, positions, sections, interleaved, dtype, eps):
    w = None if weight is None else np64(weight)
    y, size = B.norm_rotate(np64(x), w, eps, None if table is None else np64(table),
                            None if positions is None else positions.cpu().numpy(), sections, interleaved)
    rel, sub = ROUND[dtype]
    err = np.abs(np64(got) - y)
    assert got.dtype == dtype and (err <= 16 * U * size * (1 + rel) + rel * np.abs(y) + sub + 1e-37).all(), \
        float((err / (size + 1e-30)).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ROPE_CASES, ids=lambda c: "-".join(map(str, c[:4])))
def test_qk_rope_matches_the_oracle(case, dtype):
    from qsa_b200 import qsa_qk_rope

    tokens, hq, hkv, rotary, interleaved, sections, norm = case
    gen = torch.Generator().manual_seed(tokens + hq)
    # views of a packed projection
    qkv = (torch.randn(tokens, hq + 2 * max(hkv, 1), D, generator=gen) * 3).to(dtype).cuda()
    q, k = qkv[:, :hq], qkv[:, hq:hq + hkv] if hkv else None
    table = rope_table(257, rotary).cuda() if rotary else None
    axes = 1 if sections is None else len(sections)
    positions = None
    if rotary:
        positions = torch.randint(0, 257, (axes, tokens), generator=gen, dtype=torch.int32)
        positions[0, 0] = 256
        positions = positions.cuda() if axes > 1 else positions[0].cuda()
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=gen)).to(dtype).cuda() for _ in range(2)) if norm else (None, None)
    before = qkv.clone()
    q_out, k_out = qsa_qk_rope(q, k, table, positions, q_weight=wq, k_weight=wk if hkv else None, eps=1e-5,
                               interleaved=interleaved, sections=sections)
    torch.cuda.synchronize()
    assert torch.equal(qkv, before)
    _rope_check(q_out, q, wq, table, positions, sections, interleaved, dtype, 1e-5)
    if hkv:
        _rope_check(k_out, k, wk, table, positions, sections, interleaved, dtype, 1e-5)
    else:
        assert k_out is None
    # in place, on a side stream: the same bits
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        qsa_qk_rope(q, k, table, positions, q_weight=wq, k_weight=wk if hkv else None, eps=1e-5,
                    interleaved=interleaved, sections=sections, q_out=q, k_out=k)
    side.synchronize()
    assert torch.equal(q, q_out) and (not hkv or torch.equal(k, k_out))
    assert torch.equal(qkv[:, hq + hkv:], before[:, hq + hkv:])


@pytest.mark.gpu
def test_qk_rope_values_at_the_edges():
    from qsa_b200 import qsa_qk_rope

    table = rope_table(8, 64).cuda()
    x = torch.randn(6, 2, D, device="cuda")
    x[1] = 0.0
    x[2, 0, 5] = float("nan")
    x[3, 0, 70] = float("inf")
    x[4] *= 1e-25  # squares below fp32's range: eps alone
    pos = torch.tensor([0, 1, 2, 3, 4, 8], dtype=torch.int32, device="cuda")  # 8: past the table
    w = torch.ones(D, device="cuda")
    y, none = qsa_qk_rope(x, None, table, pos, q_weight=w)
    assert none is None and torch.isfinite(y[[0, 1, 4, 5]]).all()
    assert not y[1].any() and not y[5].any() and y[0].any()
    assert y[2, 0].isnan().all() and torch.isfinite(y[2, 1]).all()
    assert y[3, 0, 70].isnan() and torch.isfinite(y[3, 1]).all()
    # without a norm NaN and infinity stay in their pair
    y, _ = qsa_qk_rope(x, None, table, pos)
    assert sorted(y[2, 0].isnan().nonzero().flatten().tolist()) == [5, 37]
    assert y[3, 0, 70].isinf() and torch.isfinite(y[3, 0, :70]).all()
    y, _ = qsa_qk_rope(x, None, table, pos - 1)
    assert not y[0].any() and y[1:2].eq(0).all() and y[5].any()  # position -1; zeros; position 7


# ------------------------------------------------------------- GPU: append ----
def _caches(gen, pages, page, block, hkv):
    codes = torch.randint(0, 256, (2, pages, page, hkv, D), generator=gen, dtype=torch.uint8)
    codes[(codes & 0x7F) == 0x7F] = 0x35
    scales = torch.rand((2, pages, page // block, hkv), generator=gen) * 0.02 + 1e-3
    return codes, scales


def _check_append(got, want, cache0, scales0, x_err, s_err):
    """got (codes, scales) against the oracle's dict; x_err / s_err: error of
    the new rows' values (array like them, over s) and of the scales."""
    codes, scales = got
    tab = O.e4m3fn_table().astype(np.float64)
    touched = want["scales"] != np.asarray(scales0, np.float64)
    assert np.array_equal(scales[~touched], scales0[~touched])
    assert (np.abs(scales - want["scales"]) <= s_err * want["scales"]).all()
    written = want["written"]
    assert np.array_equal(codes[~written], cache0[~written])
    v, c = want["values"][written], tab[codes[written]]
    nan = np.isnan(v)
    assert np.array_equal(nan, np.isnan(c))
    inf = np.isinf(v)
    assert (c[inf] == np.sign(v[inf]) * 448).all()
    fin = ~nan & ~inf
    v, c, e = v[fin], c[fin], np.broadcast_to(x_err, want["values"].shape)[written][fin]
    near = np.clip(v, -448, 448)
    bad = np.abs(c - near) > np.maximum(B.step(c), B.step(near)) / 2 + e + (4 * U + s_err) * np.abs(near)
    assert not bad.any(), (c[bad][:5], v[bad][:5])


APPEND_CASES = {
    # page, block, hkv, rotary, interleaved, sections, norm, starts, counts
    "one_token_each": (16, 16, 8, 128, False, None, True, [0, 1, 15, 16, 31, 40], None),
    "per_token_scales": (8, 1, 2, 64, False, None, True, [0, 3, 7, 9], [1, 6, 2, 0]),
    "ragged": (16, 16, 3, 128, False, None, True, [0, 5, 16, 30, 2], [33, 0, 1, 18, 14]),
    "odd_blocks": (24, 12, 5, 32, True, None, True, [0, 11, 12, 37], [25, 2, 12, 40]),
    "one_scale_a_page": (64, 64, 1, 0, False, None, False, [0, 60, 63], [64, 5, 130]),
    "large_blocks": (128, 128, 2, 128, False, (16, 24, 24), True, [0, 100], [300, 29]),
    "pages_of_one": (1, 1, 2, 128, False, None, True, [0, 5, 3], [9, 1, 17]),
    "runs_over_pages": (12, 4, 3, 64, True, None, True, [0, 11, 13, 2], [30, 7, 12, 1]),
    "pairs_one_token_each": (16, 2, 9, 128, False, None, True, [0, 1, 14, 15, 17], None),
    "many_entries": (16, 8, 1, 128, False, None, True, [(7 * i) % 40 for i in range(80)], [(5 * i) % 11 for i in range(80)]),
    "blocks_past_the_held": (256, 256, 2, 128, False, None, True, [0, 200, 255], [300, 3, 70]),
    "tiny_blocks": (48, 3, 4, 16, False, (1, 7), False, [2, 0, 46], [50, 4, 5]),
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", sorted(APPEND_CASES))
def test_block_append_matches_the_oracle(name, dtype):
    from qsa_b200 import qsa_block_append

    page, block, hkv, rotary, interleaved, sections, norm, starts, counts = APPEND_CASES[name]
    gen = torch.Generator().manual_seed(len(name))
    n = len(starts)
    ppr = -(-max(s + (1 if counts is None else c) for s, c in zip(starts, counts or starts)) // page)
    pages = n * ppr + 2
    btable = torch.randperm(pages, generator=gen)[:n * ppr].view(n, ppr).to(torch.int32)
    cu = None if counts is None else np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    total = n if counts is None else int(cu[-1])
    kv = (torch.randn(total, 2 * hkv, D, generator=gen) * torch.exp(torch.randn(total, 1, 1, generator=gen))).to(dtype)
    kv[0, hkv:] = 0.0
    w = (1 + 0.3 * torch.randn(D, generator=gen)).to(dtype) if norm else None
    table = rope_table(400, rotary) if rotary else None
    positions = torch.randint(0, 400, (len(sections), total), generator=gen, dtype=torch.int32) if sections else None
    codes, scales = _caches(gen, pages, page, block, hkv)
    reqs = torch.randperm(n, generator=gen).to(torch.int32)
    kc, vc = (c.cuda().view(torch.float8_e4m3fn) for c in codes)
    ks, vs = (s.cuda() for s in scales)
    kv_d = kv.cuda()
    dev = lambda t: None if t is None else t.cuda()
    qsa_block_append(kv_d[:, :hkv], kv_d[:, hkv:], kc, vc, ks, vs, btable.cuda(),
                     torch.tensor(starts, dtype=torch.int32).cuda(), reqs=reqs.cuda(),
                     cu_tokens=None if cu is None else torch.from_numpy(cu).cuda(), table=dev(table),
                     positions=dev(positions), k_weight=dev(w), eps=1e-5, interleaved=interleaved, sections=sections)
    torch.cuda.synchronize()
    pos = np.concatenate([s + np.arange(c) for s, c in zip(starts, counts or [1] * n)])
    k, size = B.norm_rotate(np64(kv[:, :hkv]), None if w is None else np64(w), 1e-5,
                            None if table is None else np64(table), positions.numpy() if sections else pos, sections,
                            interleaved)
    want = B.append(k, np64(kv[:, hkv:]), codes[0].numpy(), codes[1].numpy(), scales[0].numpy(), scales[1].numpy(),
                    btable.numpy(), starts, reqs.numpy(), cu)
    key_err = 0.0 if not norm and not rotary else 16 * U
    # a key's error over its scale: its terms are at most sqrt(2) of the row's largest, 448 s
    _check_append((u8(kc), ks.cpu().numpy()), want[0], codes[0].numpy(), scales[0].numpy(), key_err * 2 * 448, key_err * 2 + 2 * U)
    _check_append((u8(vc), vs.cpu().numpy()), want[1], codes[1].numpy(), scales[1].numpy(), 0.0, U)


@pytest.mark.gpu
def test_block_append_skips_what_lies_outside():
    from qsa_b200 import qsa_block_append

    gen = torch.Generator().manual_seed(3)
    page, block, hkv, pages = 8, 4, 2, 12
    codes, scales = _caches(gen, pages, page, block, hkv)
    # a wide table of which two columns count; page ids outside the cache
    wide = torch.full((5, 6), 11, dtype=torch.int32)
    wide[:, 1:3] = torch.tensor([[0, 1], [2, -1], [4, 12], [6, 7], [8, 9]], dtype=torch.int32)
    starts = [6, 4, 0, -3, 14]
    counts = [12, 10, 12, 4, 5]  # past the table, onto page -1, onto page 12, negative start, past the table
    reqs = torch.tensor([0, 1, 2, 3, 5], dtype=torch.int32)  # the last one out of range
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    kv = torch.randn(int(cu[-1]), 2 * hkv, D, generator=gen)
    kc, vc = (c.cuda().view(torch.float8_e4m3fn) for c in codes)
    ks, vs = (s.cuda() for s in scales)
    kv_d = kv.cuda()
    qsa_block_append(kv_d[:, :hkv], kv_d[:, hkv:], kc, vc, ks, vs, wide.cuda()[:, 1:3],
                     torch.tensor(starts, dtype=torch.int32).cuda(), reqs=reqs.cuda(), cu_tokens=torch.from_numpy(cu).cuda())
    torch.cuda.synchronize()
    want = B.append(np64(kv[:, :hkv]), np64(kv[:, hkv:]), codes[0].numpy(), codes[1].numpy(), scales[0].numpy(),
                    scales[1].numpy(), wide[:, 1:3].numpy(), starts, reqs.numpy(), cu)
    for got, s, w, c0, s0 in ((kc, ks, want[0], codes[0], scales[0]), (vc, vs, want[1], codes[1], scales[1])):
        assert 0 < w["written"].sum() < w["written"].size
        _check_append((u8(got), s.cpu().numpy()), w, c0.numpy(), s0.numpy(), 0.0, U)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_block_append_values_at_the_edges(dtype):
    from qsa_b200 import block_cache, qsa_block_append

    hkv, page = 1, 4
    big = torch.finfo(dtype).max
    rows = torch.randn(8, 2 * hkv, D, generator=torch.Generator().manual_seed(5))
    rows[0] = 0.0                                       # a block of zeros alone
    rows[1, :, 3], rows[1, :, 4] = float("inf"), -float("inf")
    rows[2, :, 7] = float("nan")
    rows[3] = float("inf")                              # nothing finite
    rows[4, :, 0] = big
    rows[5] *= torch.finfo(dtype).tiny                  # smaller than 448 * 2^-126 in bf16 and fp32
    rows[6] = torch.linspace(-1, 1, D)
    kv = rows.to(dtype)
    kc, vc, ks, vs = block_cache(8, page, hkv, page)
    btable = torch.arange(8, dtype=torch.int32).view(8, 1)
    starts = [0] * 8
    kv_d = kv.cuda()
    qsa_block_append(kv_d[:, :1], kv_d[:, 1:], kc, vc, ks, vs, btable.cuda(), torch.zeros(8, dtype=torch.int32).cuda())
    torch.cuda.synchronize()
    zero = np.zeros((8, page, 1, D), np.uint8), np.zeros((8, 1, 1), np.float32)
    want = B.append(np64(kv[:, :1]), np64(kv[:, 1:]), zero[0], zero[0], zero[1], zero[1], btable.numpy(), starts)
    for got, s, w in ((kc, ks, want[0]), (vc, vs, want[1])):
        _check_append((u8(got), s.cpu().numpy()), w, zero[0], zero[1], 0.0, 2 * U)
    assert ks[0].item() == 2.0 ** -126 and not u8(kc)[0].any()


@pytest.mark.gpu
def test_block_append_token_by_token_holds_what_a_prompt_holds():
    """Ten tokens one by one into blocks of four: the block scales of one
    append of all ten, and rows within one more rounding of its codes."""
    from qsa_b200 import block_cache, qsa_block_append

    gen = torch.Generator().manual_seed(9)
    kv = (torch.randn(10, 4, D, generator=gen) * torch.exp(2 * torch.randn(10, 1, 1, generator=gen))).to(torch.bfloat16).cuda()
    btable = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    one, whole = block_cache(2, 8, 2, 4), block_cache(2, 8, 2, 4)
    one[0].view(torch.uint8).fill_(0x7F)  # stale NaN codes and scales of an earlier owner
    one[2].fill_(float("nan")), one[3].fill_(1e9)
    for i in range(10):
        qsa_block_append(kv[i:i + 1, :2], kv[i:i + 1, 2:], *one, btable, torch.tensor([i], dtype=torch.int32, device="cuda"))
    qsa_block_append(kv[:, :2], kv[:, 2:], *whole, btable, torch.zeros(1, dtype=torch.int32, device="cuda"),
                     cu_tokens=torch.tensor([0, 10], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    for i in (2, 3):
        assert torch.equal(one[i][1], whole[i][1]) and torch.equal(one[i][0, 0], whole[i][0, 0])
    for i, x in ((0, kv[:, :2]), (1, kv[:, 2:])):
        for c, s, steps in ((one[i], one[i + 2], 2.0), (whole[i], whole[i + 2], 0.5)):
            val = np64(c).reshape(2, 2, 4, 2, D) * np64(s)[:, :, None, :, None]
            val = val[[1, 0]].reshape(16, 2, D)[:10]
            sc = np64(s)[[1, 0]].reshape(4, 2).repeat(4, 0)[:10][..., None]
            # each growth of a scale rounds a kept code once more
            assert (np.abs(val - np64(x)) <= steps * B.step(np64(x) / sc) * sc * (1 + 1e-6)).all()


# ------------------------------------------------------------- GPU: decode ----
def _bf16(t):
    return t.to(torch.bfloat16)


def _decode_inputs(gen, rows, reqs, hq, hkv, page, block, ppr, kv_std=60.0):
    pages = reqs * ppr + 3
    q = _bf16(torch.randn(rows, hq, D, generator=gen))
    gate = _bf16(torch.randn(rows, hq, D, generator=gen))
    kv = (torch.randn(2, pages, page, hkv, D, generator=gen) * kv_std).clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = 0.02 * torch.exp2(4 * torch.rand((2, pages, page // block, hkv), generator=gen) - 2)
    btable = torch.randperm(pages, generator=gen)[:reqs * ppr].view(reqs, ppr).to(torch.int32)
    t2r = torch.randint(0, reqs, (rows,), generator=gen, dtype=torch.int32)
    return q, gate, kv[0], kv[1], scales[0], scales[1], btable, t2r


def _decode_check(out, q, k, v, ks, vs, btable, t2r, indices, counts, gate, softmax_scale=None, rows=None):
    n = lambda t: None if t is None else t.cpu().numpy()
    rows = slice(None) if rows is None else rows
    pick = lambda t: None if t is None else t[rows]
    ref, size, ssize = B.decode(np64(q[rows]), u8(k), u8(v), n(ks), n(vs), n(btable), n(pick(t2r)), n(pick(indices)),
                                n(pick(counts)), None if gate is None else np64(gate[rows]), softmax_scale)
    tol = 2.0 ** -8 * np.abs(ref) + size * (2.0 ** -10 + 2.0 ** -12 + 2 * (2.0 ** -17 * ssize)[..., None]) + 1e-37
    err = np.abs(np64(out[rows]) - ref)
    assert not np.isnan(err).any()
    assert (err <= tol).all(), (float((err / tol).max()), np.argwhere(err > tol)[:4])
    return ref


GROUPS = [(1, 8), (2, 4), (3, 3), (4, 8), (5, 5), (7, 2), (8, 8), (9, 1), (12, 3), (16, 2), (17, 2), (20, 1), (31, 1), (32, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("group,hkv", GROUPS)
@pytest.mark.parametrize("dense", [False, True])
def test_block_decode_groups_and_ragged_rows(group, hkv, dense):
    from qsa_b200 import qsa_block_decode

    gen = torch.Generator().manual_seed(group * 10 + hkv)
    rows, reqs, page, block, ppr = 9, 4, 16, 8, 13
    ctx = ppr * page
    q, gate, k, v, ks, vs, btable, t2r = _decode_inputs(gen, rows, reqs, group * hkv, hkv, page, block, ppr)
    counts = torch.tensor([0, 1, 15, 16, 17, 100, 129, ctx, ctx + 50], dtype=torch.int32)
    indices = None
    if not dense:
        indices = torch.stack([torch.randperm(ctx, generator=gen) for _ in range(rows)])[:, :150].to(torch.int32)
        indices[torch.rand(rows, 150, generator=gen) < 0.1] = -1
        indices[3] = -1                                    # every entry masked
        indices[4, :] = indices[4, 0].clamp_min(0)         # one token over and over
        indices[5, ::7] = ctx + 3                          # past the block table
        indices[6, 1::5] = 2 ** 31 - 1
    c = lambda t: None if t is None else t.cuda()
    out = qsa_block_decode(c(q), c(k), c(v), c(ks), c(vs), c(btable), c(t2r), c(indices), gate=c(gate), counts=c(counts))
    torch.cuda.synchronize()
    ref = _decode_check(out, q, k, v, ks, vs, btable, t2r, indices, counts, gate)
    assert not out[0].any() and not ref[0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("page,block", [(1, 1), (16, 16), (16, 1), (24, 12), (48, 8), (64, 64), (100, 20), (128, 128), (256, 32)])
@pytest.mark.parametrize("rows,ctx", [(1, 1), (2, 33), (3, 2500), (40, 700)])
def test_block_decode_pages_and_lengths(page, block, rows, ctx):
    from qsa_b200 import qsa_block_decode

    gen = torch.Generator().manual_seed(page * 7 + ctx)
    hkv, group = 2, 4
    ppr = -(-ctx // page)
    q, _, k, v, ks, vs, btable, t2r = _decode_inputs(gen, rows, rows, group * hkv, hkv, page, block, ppr)
    # a table inside a wider one
    wide = torch.full((rows, ppr + 5), 10 ** 9, dtype=torch.int32)
    wide[:, 2:2 + ppr] = btable
    counts = torch.randint(0, ctx + 1, (rows,), generator=gen, dtype=torch.int32)
    counts[0] = ctx
    c = lambda t: t.cuda()
    args = [c(q), c(k), c(v), c(ks), c(vs), c(wide)[:, 2:2 + ppr], None]
    out = qsa_block_decode(*args, counts=c(counts))
    again = torch.full_like(args[0], float("nan"))
    assert qsa_block_decode(*args, counts=c(counts), out=again) is again
    full = qsa_block_decode(*args, softmax_scale=0.3)
    torch.cuda.synchronize()
    assert torch.equal(out, again)  # the same bits, into a given tensor
    _decode_check(out, q, k, v, ks, vs, btable, None, None, counts, None)
    _decode_check(full, q, k, v, ks, vs, btable, None, None, None, None, softmax_scale=0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 5, 300])
def test_block_decode_long_selections(rows):
    """More columns than one CTA takes, in strided indices, some rows short."""
    from qsa_b200 import qsa_block_decode

    gen = torch.Generator().manual_seed(rows)
    hkv, group, page, block, ppr, topk = 4, 4, 16, 4, 400, 3001
    reqs = min(rows, 6)
    q, gate, k, v, ks, vs, btable, t2r = _decode_inputs(gen, rows, reqs, group * hkv, hkv, page, block, ppr)
    indices = torch.argsort(torch.rand(rows, ppr * page, generator=gen), 1)[:, :topk + 4].to(torch.int32)
    short = torch.randint(0, topk, (rows,), generator=gen)
    short[0] = topk
    indices[torch.arange(topk + 4)[None] >= short[:, None]] = -1
    view = indices.cuda()[:, :topk]
    c = lambda t: t.cuda()
    out = qsa_block_decode(c(q), c(k), c(v), c(ks), c(vs), c(btable), c(t2r), view, gate=c(gate))
    torch.cuda.synchronize()
    pick = list(range(rows)) if rows <= 5 else [0, 1, 77, 150, 298, 299]
    _decode_check(out, q, k, v, ks, vs, btable, t2r, indices[:, :topk], None, gate, rows=pick)


@pytest.mark.gpu
@pytest.mark.parametrize("dense", [False, True])
def test_block_decode_reads_nothing_that_is_masked(dense):
    """NaN codes and scales in stale rows, foreign pages and past the counts."""
    from qsa_b200 import qsa_block_decode

    gen = torch.Generator().manual_seed(21)
    rows, hkv, group, page, block, ppr = 4, 2, 8, 16, 16, 5
    q, gate, k, v, ks, vs, btable, _ = _decode_inputs(gen, rows, rows, group * hkv, hkv, page, block, ppr)
    counts = torch.tensor([37, 64, 1, 80], dtype=torch.int32)
    t2r = torch.tensor([0, 1, 2, 7], dtype=torch.int32)  # the last row's request is out of range
    btable[1, 2] = -1                                     # a page that is not there
    kb, vb = k.view(torch.uint8), v.view(torch.uint8)
    seen = torch.zeros(k.shape[0], page, dtype=torch.bool)
    for r in range(3):
        for t in range(int(counts[r])):
            if btable[r, t // page] >= 0:
                seen[btable[r, t // page], t % page] = True
    kb[~seen], vb[~seen] = 0x7F, 0xFF
    ks[~seen.any(1)], vs[~seen.any(1)] = float("nan"), float("inf")
    indices = None
    if not dense:
        indices = torch.arange(ppr * page, dtype=torch.int32).repeat(rows, 1)
        indices = torch.where(indices < counts[:, None], indices, -1)
        indices = indices[:, torch.randperm(ppr * page, generator=gen)].contiguous()
    c = lambda t: None if t is None else t.cuda()
    out = qsa_block_decode(c(q), c(k), c(v), c(ks), c(vs), c(btable), c(t2r), c(indices), gate=c(gate),
                           counts=c(counts) if dense else None)
    torch.cuda.synchronize()
    assert torch.isfinite(out).all() and not out[3].any()
    _decode_check(out, q, k, v, ks, vs, btable, t2r, indices, counts if dense else None, gate)


@pytest.mark.gpu
def test_block_decode_nan_in_a_valid_place_shows():
    from qsa_b200 import qsa_block_decode

    gen = torch.Generator().manual_seed(22)
    rows, hkv, group, page = 3, 2, 4, 16
    q, _, k, v, ks, vs, btable, _ = _decode_inputs(gen, rows, rows, group * hkv, hkv, page, page, 4)
    k.view(torch.uint8)[btable[0, 1], 3, 0, 9] = 0x7F   # row 0, head 0: every output
    v.view(torch.uint8)[btable[1, 2], 5, 1, 17] = 0x7F  # row 1, head 1: dim 17
    out = qsa_block_decode(*(t.cuda() for t in (q, k, v, ks, vs, btable)), None)
    nan = out.isnan().cpu()
    want = torch.zeros_like(nan)
    want[0, :group] = True
    want[1, group:, 17] = True
    assert torch.equal(nan, want)


@pytest.mark.gpu
@pytest.mark.parametrize("spread", ["scales", "scores", "queries"])
def test_block_decode_wide_ranges(spread):
    """Scales over many powers of two, scores far apart, uneven queries."""
    from qsa_b200 import qsa_block_decode

    gen = torch.Generator().manual_seed(23)
    rows, hkv, group, page, block, ppr = 5, 2, 6, 16, 4, 30
    q, gate, k, v, ks, vs, btable, t2r = _decode_inputs(gen, rows, rows, group * hkv, hkv, page, block, ppr)
    if spread == "scales":
        ks *= torch.exp2(torch.randint(-20, 1, ks.shape, generator=gen).float())
        vs *= torch.exp2(torch.randint(-60, 60, vs.shape, generator=gen).float())
    elif spread == "scores":
        q = _bf16(q.float() * 12)
    else:
        q[:, :, 5] *= 3000
        q[:, 1] *= 2.0 ** -90
        q[:, 2] = 0
        q[:, 3] *= 2.0 ** 40
        ks[:] = ks * 1e-3
    c = lambda t: t.cuda()
    scale = 2.0 ** -40 if spread == "queries" else None
    out = qsa_block_decode(c(q), c(k), c(v), c(ks), c(vs), c(btable), c(t2r), gate=c(gate), softmax_scale=scale)
    torch.cuda.synchronize()
    _decode_check(out, q, k, v, ks, vs, btable, t2r, None, None, gate, softmax_scale=scale)


@pytest.mark.gpu
def test_block_decode_past_32_bits_of_offset():
    """Pages beyond 4 GiB of cache."""
    from qsa_b200 import qsa_block_append, qsa_block_decode

    hkv, page = 8, 16
    pages = (5 << 30) // (page * hkv * D)
    kc, vc = (torch.empty((pages, page, hkv, D), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.full((pages, 1, hkv), float("nan"), device="cuda") for _ in range(2))
    gen = torch.Generator().manual_seed(31)
    # the pages of the table: the first, the last and those around 2 and 4 GiB
    ids = [0, pages - 1, (1 << 31) // (page * hkv * D), (1 << 32) // (page * hkv * D), (1 << 32) // (page * hkv * D) + 1]
    btable = torch.tensor([ids], dtype=torch.int32, device="cuda")
    kv = torch.randn(73, 2 * hkv, D, generator=gen).to(torch.bfloat16).cuda()
    qsa_block_append(kv[:, :hkv], kv[:, hkv:], kc, vc, ks, vs, btable, torch.zeros(1, dtype=torch.int32, device="cuda"),
                     cu_tokens=torch.tensor([0, 73], dtype=torch.int32, device="cuda"))
    q = _bf16(torch.randn(1, 32, D, generator=gen)).cuda()
    out = qsa_block_decode(q, kc, vc, ks, vs, btable, None, counts=torch.tensor([73], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    small = [t[ids].cpu() for t in (kc.view(torch.uint8), vc.view(torch.uint8), ks, vs)]
    _decode_check(out, q, *small, torch.arange(5, dtype=torch.int32)[None], None, None, torch.tensor([73]), None)
    val = np64(small[0].view(torch.float8_e4m3fn)).reshape(80, hkv, D)[:73] * np64(small[2]).reshape(5, hkv).repeat(16, 0)[:73][..., None]
    sc = np64(small[2]).reshape(5, hkv).repeat(16, 0)[:73][..., None]
    x = np64(kv[:, :hkv])
    assert (np.abs(val - x) <= 0.5 * B.step(x / sc) * sc * (1 + 1e-5)).all()


@pytest.mark.gpu
def test_block_decode_in_a_graph_and_on_a_side_stream():
    from qsa_b200 import qsa_block_append, qsa_block_decode, qsa_qk_rope

    gen = torch.Generator().manual_seed(41)
    rows, hkv, group, page, block, ppr = 6, 4, 4, 16, 16, 70
    q, gate, k, v, ks, vs, btable, t2r = (t.cuda() for t in _decode_inputs(gen, rows, rows, 16, hkv, page, block, ppr))
    t2r = torch.arange(rows, dtype=torch.int32, device="cuda")
    starts = torch.randint(0, ppr * page - 1, (rows,), generator=gen, dtype=torch.int32).cuda()
    kv = torch.randn(rows, 2 * hkv, D, generator=gen).to(torch.bfloat16).cuda()
    table = rope_table(ppr * page, 128).cuda()

    def step():
        qr, _ = qsa_qk_rope(q, None, table, starts)
        qsa_block_append(kv[:, :hkv], kv[:, hkv:], k, v, ks, vs, btable, starts, table=table)
        return qsa_block_decode(qr, k, v, ks, vs, btable, t2r, gate=gate, counts=starts + 1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        captured.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, eager)  # the same rows again: the same bits
    qr, _ = qsa_qk_rope(q, None, table, starts)
    _decode_check(eager, qr, k.cpu(), v.cpu(), ks, vs, btable, t2r, None, starts + 1, gate)


@pytest.mark.gpu
def test_operators_refuse_what_does_not_fit():
    from qsa_b200 import block_cache, qsa_block_append, qsa_block_decode, qsa_qk_rope

    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    q = torch.zeros(4, 8, D, device="cuda", dtype=torch.bfloat16)
    table = rope_table(8, 64).cuda()
    with pytest.raises(RuntimeError, match="positions"):
        qsa_qk_rope(q, None, table)
    with pytest.raises(RuntimeError, match="int32"):
        qsa_qk_rope(q, None, table, torch.zeros(4, device="cuda", dtype=torch.int64))
    with pytest.raises(RuntimeError, match="section"):
        qsa_qk_rope(q, None, table, torch.zeros(3, 4, device="cuda", dtype=torch.int32))
    with pytest.raises(RuntimeError, match="head_dim|unsupported"):
        qsa_qk_rope(q[..., :64].contiguous())
    with pytest.raises(RuntimeError, match="dtype"):
        qsa_qk_rope(q, q.float(), table, i32(0, 0, 0, 0))
    with pytest.raises(NotImplementedError):
        qsa_qk_rope(q.cpu())
    caches = block_cache(4, 16, 2, 16)
    bt = i32(0, 1, 2, 3).view(2, 2)
    kv = torch.zeros(2, 2, D, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="one token"):
        qsa_block_append(kv, kv, *caches, bt, i32(0))
    with pytest.raises(RuntimeError, match="v_new"):
        qsa_block_append(kv, kv.float(), *caches, bt, i32(0, 0))
    with pytest.raises(RuntimeError, match="cu_tokens"):
        qsa_block_append(kv, kv, *caches, bt, i32(0, 0), cu_tokens=i32(0, 2))
    with pytest.raises(RuntimeError, match="blocks"):
        qsa_block_append(kv, kv, *caches[:2], *(torch.zeros(4, 3, 2, device="cuda") for _ in range(2)), bt, i32(0, 0))
    with pytest.raises(RuntimeError, match="bfloat16"):
        qsa_block_decode(q.float(), *caches, bt, i32(0, 0, 1, 1))
    with pytest.raises(RuntimeError, match="t2r"):
        qsa_block_decode(q, *caches, bt, i32(0, 0))
    with pytest.raises(RuntimeError, match="group"):
        qsa_block_decode(torch.zeros(4, 66, D, device="cuda", dtype=torch.bfloat16), *caches, bt, None)
    with pytest.raises(RuntimeError, match="sizes|unsupported"):
        qsa_block_decode(q[:, :7].contiguous(), *caches, bt, None)
    assert qsa_block_decode(q[:0], *caches, bt, None).shape == (0, 8, D)
    none = torch.empty(4, 0, dtype=torch.int32, device="cuda")
    assert not qsa_block_decode(q, *caches, bt, i32(0, 0, 1, 1), none).any()


@pytest.mark.gpu
def test_the_serving_example_runs_the_operators_together():
    """Against fp32 from the projections, so with the codes' own error: a value
    is off by up to 2^-4 of itself (2^-4 / sqrt(3) / 2 or so on average) and a
    score by the same of |q||k| / sqrt(128), of some tens of terms."""
    import importlib.util

    from conftest import REPO

    spec = importlib.util.spec_from_file_location("block_cache_serving", REPO / "examples" / "block_cache_serving.py")
    example = importlib.util.module_from_spec(spec)
    import sys

    sys.modules[spec.name] = example
    spec.loader.exec_module(example)
    for kw in (dict(), dict(requests=3, steps=2, hq=12, hkv=2, page=24, block=8, topk=7, seed=1)):
        dense, sparse = example.serve(**kw)
        assert dense < 0.08 and sparse < 0.08, (dense, sparse)


@pytest.mark.gpu
@pytest.mark.parametrize("group,hkv", [(1, 8), (8, 1), (5, 3), (4, 6), (12, 2), (16, 4), (9, 1), (20, 1), (32, 2), (17, 8)])
@pytest.mark.parametrize("dense", [False, True])
def test_block_decode_planned_rows(group, hkv, dense):
    """Rows of more than 512 columns: shared evenly by the GPU's CTAs, cut and
    joined, for every layout of heads; empty and short rows between long ones."""
    from qsa_b200 import qsa_block_decode

    gen = torch.Generator().manual_seed(100 * group + hkv)
    rows, reqs, page, block, ppr = 7, 3, 16, 4, 130
    ctx = ppr * page
    q, gate, k, v, ks, vs, btable, t2r = _decode_inputs(gen, rows, reqs, group * hkv, hkv, page, block, ppr)
    counts = torch.tensor([1501, 0, 1, ctx, 17, 0, 777], dtype=torch.int32)
    indices = None
    if not dense:
        indices = torch.argsort(torch.rand(rows, ctx, generator=gen), 1)[:, :1600].to(torch.int32)
        indices[torch.rand(rows, 1600, generator=gen) < 0.02] = -1
        indices[4] = -1
    c = lambda t: None if t is None else t.cuda()
    args = [c(t) for t in (q, k, v, ks, vs, btable, t2r, indices)]
    out = qsa_block_decode(*args, gate=c(gate), counts=c(counts))
    again = qsa_block_decode(*args, gate=c(gate), counts=c(counts))
    torch.cuda.synchronize()
    assert torch.equal(out, again)
    _decode_check(out, q, k, v, ks, vs, btable, t2r, indices, counts, gate)
    assert not out[1].any() and not out[5].any()


@pytest.mark.gpu
@pytest.mark.parametrize("group,hkv", [(4, 8), (3, 1), (10, 2)])
def test_block_decode_one_long_row_in_many_pieces(group, hkv):
    from qsa_b200 import qsa_block_decode

    gen = torch.Generator().manual_seed(group)
    page, ppr = 64, 130
    q, gate, k, v, ks, vs, btable, _ = _decode_inputs(gen, 2, 2, group * hkv, hkv, page, page, ppr)
    counts = torch.tensor([8317, 3], dtype=torch.int32)
    c = lambda t: t.cuda()
    out = qsa_block_decode(c(q), c(k), c(v), c(ks), c(vs), c(btable), None, gate=c(gate), counts=c(counts))
    torch.cuda.synchronize()
    _decode_check(out, q, k, v, ks, vs, btable, None, None, counts, gate)


@pytest.mark.gpu
def test_c_abi_calls_with_a_callers_workspace():
    """The C entry points on raw pointers: the torch operators' results, and
    refusals of a missing, small or misaligned workspace."""
    from qsa_b200 import capi, qsa_block_decode, qsa_qk_rope

    gen = torch.Generator().manual_seed(51)
    rows, hkv, group, page, ppr = 3, 2, 4, 16, 60
    q, gate, k, v, ks, vs, btable, _ = (t.cuda() for t in _decode_inputs(gen, rows, rows, 8, hkv, page, page, ppr))
    counts = torch.tensor([950, 0, 600], dtype=torch.int32, device="cuda")
    want = qsa_block_decode(q, k, v, ks, vs, btable, None, gate=gate, counts=counts)
    out = torch.empty_like(q)
    ptr = lambda t: ctypes.c_void_p(t.data_ptr())
    a = capi.BlockDecodeArgs(q=ptr(q), k_cache=ptr(k), v_cache=ptr(v), k_scales=ptr(ks), v_scales=ptr(vs), counts=ptr(counts),
                             btable=ptr(btable), gate=ptr(gate), out=ptr(out), softmax_scale=D ** -0.5, rows=rows,
                             num_q_heads=8, num_kv_heads=hkv, head_dim=D, page_size=page, block_size=page,
                             pages_per_req=ppr, num_reqs=rows, num_pages=k.shape[0], btable_stride=ppr)
    need = capi.block_decode_workspace_bytes(a)
    assert need > 0
    ws = torch.randint(0, 256, (need + 256,), dtype=torch.uint8, device="cuda")  # needs no clearing
    stream = torch.cuda.current_stream().cuda_stream
    assert capi.block_decode(a, None, 0, stream) == capi.ERR_WORKSPACE
    assert capi.block_decode(a, ws, need - 1, stream) == capi.ERR_WORKSPACE
    assert capi.block_decode(a, ws[16:], need, stream) == capi.ERR_MISALIGNED
    for _ in range(2):
        assert capi.block_decode(a, ws, need, stream) == capi.OK
    torch.cuda.synchronize()
    assert torch.equal(out, want)

    table = rope_table(1000, 128).cuda()
    y = torch.empty_like(q)
    r = capi.QkRopeArgs(q=ptr(q), q_out=ptr(y), tokens=rows, num_q_heads=8, head_dim=D, q_stride=8 * D, q_out_stride=8 * D,
                        dtype=capi.DTYPE_BF16)
    r.rope.table, r.rope.positions = ptr(table), ptr(counts)
    r.rope.table_len, r.rope.rotary_dim, r.rope.num_axes = 1000, 128, 1
    assert capi.qk_rope(r, stream) == capi.OK
    want, _ = qsa_qk_rope(q, None, table, counts)
    torch.cuda.synchronize()
    assert torch.equal(y, want)


@pytest.mark.gpu
def test_strides_that_break_a_vector_load_are_refused():
    from qsa_b200 import block_cache, qsa_block_append, qsa_qk_rope

    wide = torch.zeros(4, 2 * D + 4, device="cuda", dtype=torch.bfloat16)
    x = wide[:, :2 * D].unflatten(1, (2, D))  # token stride 260 elements: 520 bytes
    with pytest.raises(RuntimeError, match="aligned"):
        qsa_qk_rope(x)
    with pytest.raises(RuntimeError, match="aligned"):
        qsa_block_append(x, x, *block_cache(4, 4, 2), torch.zeros(4, 1, device="cuda", dtype=torch.int32),
                         torch.zeros(4, device="cuda", dtype=torch.int32))
    with pytest.raises(RuntimeError, match="contiguous heads"):
        qsa_qk_rope(torch.zeros(4, D, 2, device="cuda").transpose(1, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("group,hkv", [(16, 8), (12, 4), (9, 2), (11, 1), (17, 8), (32, 2), (20, 1), (31, 4)])
@pytest.mark.parametrize("columns", [500, 1900])
def test_block_decode_wide_groups_over_much_work(group, hkv, columns):
    """Enough work for a warp to take 16 query heads (2^19 rows, columns and KV
    heads): some of the rows, the first and the last among them."""
    from qsa_b200 import qsa_block_decode

    gen = torch.Generator().manual_seed(group + columns)
    rows, reqs, page, block, ppr = (1 << 19) // (hkv * columns) + 2, 3, 16, 8, 125
    q, gate, k, v, ks, vs, btable, t2r = _decode_inputs(gen, rows, reqs, group * hkv, hkv, page, block, ppr)
    indices = torch.randint(0, ppr * page, (rows, columns), generator=gen, dtype=torch.int32)
    counts = torch.randint(0, columns + 1, (rows,), generator=gen, dtype=torch.int32)
    counts[0], counts[1], counts[-1] = columns, 0, 33
    c = lambda t: t.cuda()
    out = qsa_block_decode(*(c(t) for t in (q, k, v, ks, vs, btable, t2r, indices)), gate=c(gate), counts=c(counts))
    torch.cuda.synchronize()
    pick = [0, 1, rows // 3, rows // 2, rows - 1]
    _decode_check(out, q, k, v, ks, vs, btable, t2r, indices, counts, gate, rows=pick)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hkv", [5, 8])
@pytest.mark.parametrize("page,block", [(16, 1), (16, 2), (12, 4), (16, 16), (64, 64), (128, 128)])
def test_block_append_of_much_work_holds_what_small_calls_hold(page, block, hkv, dtype):
    """A large call, whose warps go through several heads of a block, against a
    call for each request, whose warps take one: the same bits."""
    from qsa_b200 import qsa_block_append

    gen = torch.Generator().manual_seed(page + block + hkv)
    n = 40
    counts = torch.randint(1, 600, (n,), generator=gen)
    starts = torch.randint(0, 90, (n,), generator=gen).to(torch.int32).cuda()
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).to(torch.int32)
    ppr = -(-700 // page)
    pages = n * ppr
    btable = torch.randperm(pages, generator=gen).view(n, ppr).to(torch.int32).cuda()
    kv = torch.randn(int(cu[-1]), 2 * hkv, D, generator=gen).to(dtype).cuda()
    w = (1 + 0.3 * torch.randn(D, generator=gen)).to(dtype).cuda()
    table = rope_table(700, 64).cuda()
    codes, scales = _caches(gen, pages, page, block, hkv)
    results = []
    for parts in ([(0, n)], [(e, e + 1) for e in range(n)]):
        kc, vc = (c.clone().cuda().view(torch.float8_e4m3fn) for c in codes)
        ks, vs = (s.clone().cuda() for s in scales)
        for a, b in parts:
            x = kv[int(cu[a]):int(cu[b])]
            qsa_block_append(x[:, :hkv], x[:, hkv:], kc, vc, ks, vs, btable, starts[a:b].clone(),
                             reqs=torch.arange(a, b, dtype=torch.int32, device="cuda"),
                             cu_tokens=(cu[a:b + 1] - cu[a]).cuda(), table=table, k_weight=w)
        results.append([u8(kc), u8(vc), ks.cpu().numpy(), vs.cpu().numpy()])
    for large, small in zip(*results):
        assert np.array_equal(large, small)
    assert not np.array_equal(results[0][0], codes[0].numpy())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,hq,hkv,rotary,interleaved,norm", [
    (2101, 32, 8, 128, False, True), (30011, 5, 3, 64, False, True), (12007, 13, 0, 128, True, True),
    (9001, 17, 1, 32, True, False), (6007, 24, 4, 0, False, True)])
def test_qk_rope_of_much_work_gives_what_small_calls_give(tokens, hq, hkv, rotary, interleaved, norm, dtype):
    """A large call, whose half warps go through several heads of a token,
    against calls on slices, whose half warps take one: the same bits."""
    from qsa_b200 import qsa_qk_rope

    gen = torch.Generator(device="cuda").manual_seed(tokens)
    qkv = torch.randn(tokens, hq + hkv, D, generator=gen, device="cuda").to(dtype)
    k = qkv[:, hq:] if hkv else None
    w = (1 + 0.3 * torch.randn(D, generator=gen, device="cuda")).to(dtype) if norm else None
    table = rope_table(512, rotary).cuda() if rotary else None
    positions = torch.randint(-1, 513, (tokens,), generator=gen, device="cuda", dtype=torch.int32) if rotary else None
    opts = dict(q_weight=w, interleaved=interleaved)
    large = qsa_qk_rope(qkv[:, :hq], k, table, positions, **opts)
    step = 18000 // (hq + hkv)
    for a in range(0, tokens, step):
        at = slice(a, min(a + step, tokens))
        small = qsa_qk_rope(qkv[at, :hq], None if k is None else k[at], table,
                            None if positions is None else positions[at].clone(), **opts)
        for x, y in zip(large, small):
            assert (x is None and y is None) or torch.equal(x[at], y)


# ------------------------------------- GPU: what the writer stores, attended ----
# tokens of each request, and the ranges of them whose values are zero
ZERO_CONTEXTS = [(1, [(0, 1)]), (40, [(0, 40)]), (46, [(0, 16)]), (114, [(0, 64)]), (228, [(0, 128)]), (150, [(134, 150)]),
                 (33, [(32, 33)]), (505, [(0, 256), (300, 505)]), (7, [(0, 5)])]


@pytest.mark.gpu
@pytest.mark.parametrize("group,hkv", [(4, 8), (4, 1), (3, 2), (20, 1), (12, 2), (16, 8)])
@pytest.mark.parametrize("page,block", [(16, 16), (8, 1)])
@pytest.mark.parametrize("columns", [512, 800, "two sets"])
@pytest.mark.parametrize("dense", [False, True])
def test_zero_values_appended_and_attended(group, hkv, page, block, columns, dense):
    """Values of zero get the writer's smallest scale, 2^-126: their average
    is zero, and beside other values they only count in the softmax's sum. Every
    second KV head keeps ordinary values."""
    from qsa_b200 import block_cache, qsa_block_append, qsa_block_decode

    gen = torch.Generator().manual_seed(group + hkv + page)
    counts = [n for n, _ in ZERO_CONTEXTS]
    rows = len(counts)
    used = -(-max(counts) // page)
    if columns == "two sets":  # from 2^19 (row, column, KV head)s on a warp takes 16 query heads
        columns = (1 << 19) // (rows * hkv) + page
    ppr = -(-columns // page)
    btable = torch.full((rows, ppr), -1, dtype=torch.int32)
    btable[:, :used] = torch.randperm(rows * used, generator=gen).view(rows, used).to(torch.int32)
    kv = torch.randn(sum(counts), 2 * hkv, D, generator=gen)
    at = 0
    for n, zeros in ZERO_CONTEXTS:
        for a, b in zeros:
            kv[at + a:at + b, hkv::2] = 0.0
        at += n
    kv = kv.to(torch.bfloat16).cuda()
    cache = block_cache(rows * used, page, hkv, block)
    cu = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")
    qsa_block_append(kv[:, :hkv], kv[:, hkv:], *cache, btable.cuda(), torch.zeros(rows, dtype=torch.int32, device="cuda"),
                     cu_tokens=cu)
    assert (cache[3] == 2.0 ** -126).any()
    q = _bf16(torch.randn(rows, group * hkv, D, generator=gen))
    gate = _bf16(torch.randn(rows, group * hkv, D, generator=gen))
    n = torch.tensor(counts, dtype=torch.int32)
    indices = None
    if not dense:
        indices = torch.arange(columns, dtype=torch.int32).repeat(rows, 1)
        indices = torch.where(indices < n[:, None], indices, -1)
    out = qsa_block_decode(q.cuda(), *cache, btable.cuda(), None, None if dense else indices.cuda(), gate=gate.cuda(),
                           counts=n.cuda() if dense else None)
    torch.cuda.synchronize()
    ref = _decode_check(out, q, *(t.cpu() for t in cache), btable, None, None if dense else indices[:, :max(counts)],
                        n if dense else None, gate)
    zero = (ref == 0).all(-1)
    assert zero[:2, :group].all() and not out.cpu()[torch.from_numpy(zero)].any()


@pytest.mark.gpu
@pytest.mark.parametrize("group,hkv", [(4, 8), (5, 1), (16, 8), (20, 2)])
@pytest.mark.parametrize("columns", [512, 800])
def test_block_decode_value_scales_from_zero_to_large(group, hkv, columns):
    """Value scales of 0, 2^-126 and 2^-121 beside ordinary and large ones, a
    tiny one in front of every row, and rows of tiny ones alone."""
    from qsa_b200 import qsa_block_decode

    gen = torch.Generator().manual_seed(group + hkv)
    rows, page = 8, 16
    ppr = columns // page
    q, gate, k, v, ks, vs, btable, _ = _decode_inputs(gen, rows, rows, group * hkv, hkv, page, page, ppr)
    choice = torch.tensor([0.0, 2.0 ** -126, 2.0 ** -121, 2.0 ** -100, 0.02, 8.0, 300.0])
    vs = choice[torch.randint(0, len(choice), vs.shape, generator=gen)]
    first = btable[:, 0].long()
    vs[first] = choice[torch.randint(0, 3, (rows, 1, hkv), generator=gen)]
    vs[btable[6].long()], vs[btable[7].long()] = 2.0 ** -126, 2.0 ** -121
    counts = torch.tensor([1, 16, 17, 40, 200, columns, columns - 3, 130], dtype=torch.int32)
    c = lambda t: t.cuda()
    out = qsa_block_decode(c(q), c(k), c(v), c(ks), c(vs), c(btable), None, gate=c(gate), counts=c(counts))
    torch.cuda.synchronize()
    _decode_check(out, q, k, v, ks, vs, btable, None, None, counts, gate)


@pytest.mark.gpu
@pytest.mark.parametrize("group,hkv", [(4, 8), (5, 1), (16, 8), (20, 2)])
@pytest.mark.parametrize("columns", [512, 800])
@pytest.mark.parametrize("tiny", [0.0, 2.0 ** -126])
def test_block_decode_a_large_scale_of_no_probability(group, hkv, columns, tiny):
    """Tokens whose scores lie some 300 powers of two below the others' have
    the probability 0, whatever the scale of their values."""
    from qsa_b200 import qsa_block_decode

    gen = torch.Generator().manual_seed(group + hkv)
    rows, page = 4, 16
    ppr = columns // page
    q, gate, k, v, ks, vs, btable, _ = _decode_inputs(gen, rows, rows, group * hkv, hkv, page, page, ppr)
    # along dim 0 a query of 2000 meets +-32 * 0.02: scores of about +-113, 163 powers of two either way
    q[..., 0] = 2000.0
    k[..., 0] = -32.0
    ks[:] = 0.02
    vs[:] = 1024.0
    first = btable[:, :1].long()
    k[first, :, :, 0] = 32.0
    vs[first] = tiny
    counts = torch.tensor([16, 17, 200, columns], dtype=torch.int32)
    c = lambda t: t.cuda()
    out = qsa_block_decode(c(q), c(k), c(v), c(ks), c(vs), c(btable), None, gate=c(gate), counts=c(counts))
    torch.cuda.synchronize()
    _decode_check(out, q, k, v, ks, vs, btable, None, None, counts, gate)
    assert tiny > 0 or not out.any()


def test_block_decode_refuses_columns_past_its_counters():
    """Columns are counted in int32, 2048 at a time, and so are the tiles of a
    row over its KV heads: what would overflow is refused, the largest is not."""
    from qsa_b200 import capi

    ppr = (2 ** 31 - 2048) // 16
    for over, ok in [
        (dict(indices=None, pages_per_req=ppr, btable_stride=ppr), False),  # 2^31 - 2048 columns
        (dict(indices=None, pages_per_req=ppr - 1, btable_stride=ppr), True),
        (dict(topk=2 ** 31 - 1, indices_stride=2 ** 31 - 1), False),
        (dict(topk=2 ** 31 - 2048, indices_stride=2 ** 31 - 1), False),
        (dict(topk=2 ** 31 - 2049, indices_stride=2 ** 31 - 1), True),
        (dict(topk=2 ** 30, indices_stride=2 ** 30, num_q_heads=128, num_kv_heads=128), False),
        (dict(topk=2 ** 30, indices_stride=2 ** 30, num_q_heads=63, num_kv_heads=63), True),
    ]:
        need = capi.block_decode_workspace_bytes(_decode_args(**over))
        assert need > 0 if ok else need == capi.ERR_UNSUPPORTED, (over, need)
        if not ok:
            assert capi.block_decode(_decode_args(**over)) == capi.ERR_UNSUPPORTED


def test_block_operators_refuse_heads_past_32_bits():
    """A token's heads are counted in int32 elements: up to 2^24 - 1 of them."""
    from qsa_b200 import capi

    n, stride = 1 << 24, 1 << 31
    assert capi.qk_rope(_rope_args(num_q_heads=n, q_stride=stride, q_out_stride=stride)) == capi.ERR_UNSUPPORTED
    assert capi.qk_rope(_rope_args(num_kv_heads=n, k_stride=stride, k_out_stride=stride)) == capi.ERR_UNSUPPORTED
    assert capi.qk_rope(_rope_args(num_q_heads=n - 1, q_stride=stride, q_out_stride=stride, tokens=0)) == capi.OK
    assert capi.block_append(_append_args(num_kv_heads=n, token_stride=stride)) == capi.ERR_UNSUPPORTED
    assert capi.block_append(_append_args(num_kv_heads=n - 1, token_stride=stride, tokens=0)) == capi.OK
    assert capi.block_decode(_decode_args(num_q_heads=n, num_kv_heads=n)) == capi.ERR_UNSUPPORTED
    assert capi.block_decode_workspace_bytes(_decode_args(num_q_heads=n - 1, num_kv_heads=n - 1)) == 0


def _edge_rows(gen, cu, hkv, dtype, with_max):
    """New rows [tokens, hkv, 128] of an append: in about a third of the (entry,
    head)s some rows hold infinities, NaN, zeros, the type's largest value or
    values near its smallest normal one."""
    total = int(cu[-1])
    x = torch.randn(total, hkv, D, generator=gen)
    info = torch.finfo(dtype)
    for e in range(len(cu) - 1):
        for g in range(hkv):
            if torch.rand((), generator=gen) > 0.35:
                continue
            for t in range(int(cu[e]), int(cu[e + 1])):
                if torch.rand((), generator=gen) > 0.2:
                    continue
                kind, d = (int(torch.randint(0, n, (), generator=gen)) for n in (7 if with_max else 6, D))
                if kind == 0:
                    x[t, g, d] = float("inf")
                elif kind == 1:
                    x[t, g, d], x[t, g, (d + 5) % D] = -float("inf"), float("inf")
                elif kind == 2:
                    x[t, g, d] = float("nan")
                elif kind == 3:
                    x[t, g] = float("inf")
                elif kind == 4:
                    x[t, g] = 0.0
                elif kind == 5:
                    x[t, g] *= info.tiny
                else:
                    x[t, g, d] = info.max
    return x.to(dtype)


# page, block, entries of a large call (whose warps go through several heads), most tokens of an entry
EDGE_FORMS = [(8, 1, 260, 12), (16, 2, 260, 12), (12, 4, 260, 12), (16, 16, 160, 40), (64, 64, 40, 90), (256, 256, 38, 300)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page,block,many,longest", EDGE_FORMS)
@pytest.mark.parametrize("large", [False, True])
@pytest.mark.parametrize("turned", ["plain", "rotated", "normed"])
def test_block_append_edge_values_in_every_form(page, block, many, longest, large, turned, dtype):
    """Infinities, NaN, zeros and extremes among the new rows of a call with
    cu_tokens, in some heads of some blocks, and NaN among the kept codes."""
    from qsa_b200 import qsa_block_append

    gen = torch.Generator().manual_seed(1000 * block + 10 * large + len(turned))
    hkv, n = (8, many) if large else (3, 24)
    counts = torch.randint(0, longest + 1, (n,), generator=gen)
    if block > 64 and large:  # mostly short, so that the 64-bit check stays quick
        counts = torch.where(torch.rand(n, generator=gen) < 0.85, counts % 7, counts)
    starts = torch.randint(0, 2 * block, (n,), generator=gen)
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).to(torch.int32)
    ppr = -(-(2 * block + longest) // page)
    pages = n * ppr
    btable = torch.randperm(pages, generator=gen).view(n, ppr).to(torch.int32)
    k_new = _edge_rows(gen, cu, hkv, dtype, turned != "normed")  # squares of the largest values pass fp32
    v_new = _edge_rows(gen, cu, hkv, dtype, True)
    w = (1 + 0.3 * torch.randn(D, generator=gen)).to(dtype) if turned == "normed" else None
    table = None if turned == "plain" else rope_table(2 * block + longest, 64 if turned == "normed" else D)
    codes, scales = _caches(gen, pages, page, block, hkv)
    for e in range(n):
        for t in range(int(starts[e]) - int(starts[e]) % block, int(starts[e])):
            if torch.rand((), generator=gen) < 0.2:
                codes[:, btable[e, t // page], t % page, int(torch.randint(0, hkv, (), generator=gen)), t % D] = 0x7F + 0x80 * (t % 2)
    kc, vc = (c.cuda().view(torch.float8_e4m3fn) for c in codes)
    ks, vs = (s.cuda() for s in scales)
    kv = torch.cat([k_new, v_new], 1).cuda()
    dev = lambda t: None if t is None else t.cuda()
    qsa_block_append(kv[:, :hkv], kv[:, hkv:], kc, vc, ks, vs, btable.cuda(), starts.to(torch.int32).cuda(),
                     cu_tokens=cu.cuda(), table=dev(table), k_weight=dev(w), eps=1e-5)
    torch.cuda.synchronize()
    pos = np.concatenate([np.arange(s, s + c) for s, c in zip(starts.tolist(), counts.tolist())])
    with np.errstate(invalid="ignore"):
        k, _ = B.norm_rotate(np64(k_new), None if w is None else np64(w), 1e-5, None if table is None else np64(table), pos)
        want = B.append(k, np64(v_new), codes[0].numpy(), codes[1].numpy(), scales[0].numpy(), scales[1].numpy(),
                        btable.numpy(), starts.tolist(), None, cu.numpy())
    for side in want:
        assert np.isnan(side["values"][side["written"]]).any()
    assert np.isinf(want[1]["values"][want[1]["written"]]).any()
    # as in the test of ordinary values
    key_err = 0.0 if turned == "plain" else 16 * U
    _check_append((u8(kc), ks.cpu().numpy()), want[0], codes[0].numpy(), scales[0].numpy(), key_err * 2 * 448, key_err * 2 + 2 * U)
    _check_append((u8(vc), vs.cpu().numpy()), want[1], codes[1].numpy(), scales[1].numpy(), 0.0, 2 * U)
