"""The latent cache: qsa_latent_append, qsa_latent_read, qsa_latent_decode,
qsa_latent_prefill.

CPU: the 64-bit oracle against hand-made values, and the C ABI's refusals
(they run before any device is touched). GPU: each operator against the oracle
at the sizes, masks and values where it can go wrong, and all of them together.

Tolerances, with u = 2^-24 the fp32 rounding:

* append: a normed element has 20 roundings of the sum of squares at most
  (16 products in a lane, 5 exchanges), halved by the root, 2 of the root, 2
  products: under 16 u. A code is the nearest to y / scale, off by half a step
  and 16 u of it. A rotated element is two products and a sum, 4 u of its
  terms, then one bf16 rounding (2^-8). A scale is exact, but where the norm
  leaves the largest |y| within 16 u of a power's border.
* read: one rounding to the output's type.
* decode: scores accumulate up to 576 products in fp32 (under 2^-14 of the
  size of their terms, which moves a weight by as much); queries may be split
  into terms that leave out 2^-21 of the head's largest value, and then lose
  at most as much of a score as the sum over 576 values, 2^-14 of the score's
  terms where values are as spread as here. Weights may be rounded to 8 bits
  (2^-8) in the sum of values and in the sum of weights, and, below 2^-8 of the
  largest weight on the codes, to steps of 2^-15 of it, an error of 2^-16;
  then one bf16 rounding (2^-8).
* prefill: scores accumulate 192 products; weights are rounded to the inputs'
  type (2^-8 for bf16, 2^-11 for fp16) in the sum of values; 2^-12 for the
  sums and exponentials; then one rounding to the type.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import latent_oracle as L
from oracle import qsa_oracle as O

U = 2.0 ** -24
ROUND = {torch.float32: (U, 2.0 ** -149), torch.float16: (2.0 ** -11, 2.0 ** -25), torch.bfloat16: (2.0 ** -8, 2.0 ** -133)}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
RANKS = [128, 256, 384, 512]


def np64(t):
    return t.detach().double().cpu().numpy()


def u8(t):
    return t.detach().view(torch.uint8).cpu().numpy()


# ------------------------------------------------------------------- CPU ----
def test_oracle_exponent_at_the_borders():
    top = np.array([0.0, 448.0, np.nextafter(np.float32(448), np.float32(449)), 224.0, 1.0, 2.0 ** 100, 2.0 ** -100])
    assert L.exponent(top).tolist() == [-60, 0, 1, -1, -8, 60, -60]


def test_oracle_trees_chains_and_averages():
    chain = L.visible(3, None, 6, 5)
    assert chain.tolist() == [[1, 1, 1, 0, 0, 0], [1, 1, 1, 1, 0, 0], [1, 1, 1, 1, 1, 0]]
    tree = np.array([[0b001], [0b011], [0b101]])
    assert L.visible(3, tree, 6, 5).tolist() == [[1, 1, 1, 0, 0, 0], [1, 1, 1, 1, 0, 0], [1, 1, 1, 0, 1, 0]]
    codes = np.zeros((1, 4, 128), np.uint8)
    codes[0, 1:, 0] = 0x38  # 1.0
    q = np.zeros((1, 1, 1, 192))
    got = L.decode(q, codes, np.zeros((1, 4, 64)), np.full((1, 4), 2.0), np.array([[0]]), counts=[4])
    assert got[0]["out"][0, 0, 0] == 1.5 and got[0]["size"][0, 0, 0] == 1.5
    assert L.decode(q, codes, np.zeros((1, 4, 64)), np.ones((1, 4)), np.array([[0]]), counts=[0]) == [None]


def _set(a, **over):
    for k, v in over.items():
        setattr(a.cache if hasattr(getattr(a, "cache", None), k) and not hasattr(a, k) else a, k, v)
    return a


def _cache():
    from qsa_b200 import capi

    c = capi.LatentCache()
    c.codes, c.rope, c.scales, c.btable = (ctypes.c_void_p(0x100000 * (i + 1)) for i in range(4))
    c.rank, c.rope_dim, c.page_size, c.pages_per_req, c.num_reqs, c.num_pages, c.btable_stride = 512, 64, 16, 4, 2, 8, 4
    return c


CACHE_REFUSALS = [
    (dict(rank=576), "UNSUPPORTED"), (dict(rank=0), "UNSUPPORTED"), (dict(rank=200), "UNSUPPORTED"),
    (dict(rope_dim=32), "UNSUPPORTED"), (dict(page_size=0), "BAD_SHAPE"), (dict(num_reqs=0), "BAD_SHAPE"),
    (dict(num_pages=0), "BAD_SHAPE"), (dict(btable_stride=3), "BAD_SHAPE"), (dict(pages_per_req=0), "BAD_SHAPE"),
    (dict(num_pages=1 << 27), "UNSUPPORTED"), (dict(pages_per_req=1 << 27, btable_stride=1 << 27), "UNSUPPORTED"),
    (dict(codes=None), "NULL_POINTER"), (dict(scales=None), "NULL_POINTER"), (dict(btable=None), "NULL_POINTER"),
    (dict(codes=ctypes.c_void_p(0x100008)), "MISALIGNED"), (dict(rope=ctypes.c_void_p(0x100008)), "MISALIGNED"),
]


def _append_args(**over):
    from qsa_b200 import capi

    a = capi.LatentAppendArgs()
    a.cache = _cache()
    a.c, a.r, a.starts, a.cu_tokens, a.c_weight = (ctypes.c_void_p(0x10000 * (i + 1)) for i in range(5))
    a.eps, a.entries, a.tokens, a.c_stride, a.r_stride = 1e-6, 2, 5, 576, 576
    a.rotation.table, a.rotation.table_len, a.rotation.rotary_dim, a.rotation.num_axes = ctypes.c_void_p(0x90000), 9, 64, 1
    return _set(a, **over)


def _rotation(**over):
    a = _append_args()
    return dict(rotation=_set(a.rotation, **over))


@pytest.mark.parametrize("over,want", CACHE_REFUSALS + [
    (dict(entries=-1), "BAD_SHAPE"), (dict(cu_tokens=None), "BAD_SHAPE"), (dict(starts=None), "NULL_POINTER"),
    (dict(starts=ctypes.c_void_p(0x10002)), "MISALIGNED"), (dict(input_dtype=3), "UNSUPPORTED"),
    (dict(weight_dtype=-1), "UNSUPPORTED"), (dict(eps=-1.0), "BAD_VALUE"), (dict(eps=float("inf")), "BAD_VALUE"),
    (dict(c_stride=511), "BAD_SHAPE"), (dict(r_stride=63), "BAD_SHAPE"), (dict(c=None), "NULL_POINTER"),
    (dict(r=None), "NULL_POINTER"), (dict(c_stride=580), "MISALIGNED"), (dict(r=ctypes.c_void_p(0x20008)), "MISALIGNED"),
    (dict(c_weight=ctypes.c_void_p(0x50004)), "MISALIGNED"),
    (_rotation(rotary_dim=128), "UNSUPPORTED"), (_rotation(rotary_dim=24), "UNSUPPORTED"),
    (_rotation(num_axes=2), "UNSUPPORTED"), (_rotation(table_len=0), "BAD_SHAPE"),
    (_rotation(table=ctypes.c_void_p(0x90008)), "MISALIGNED"),
])
def test_latent_append_refuses_bad_arguments_before_the_device(over, want):
    from qsa_b200 import capi

    assert capi.latent_append(_append_args(**over)) == getattr(capi, "ERR_" + want)


@pytest.mark.parametrize("over,want", CACHE_REFUSALS + [
    (dict(tokens=-1), "BAD_SHAPE"), (dict(cu_tokens=None), "BAD_SHAPE"), (dict(output_dtype=7), "UNSUPPORTED"),
    (dict(c=None), "NULL_POINTER"), (dict(r=ctypes.c_void_p(0x20004)), "MISALIGNED"),
])
def test_latent_read_refuses_bad_arguments_before_the_device(over, want):
    from qsa_b200 import capi

    a = capi.LatentReadArgs()
    a.cache = _cache()
    a.c, a.r, a.starts, a.cu_tokens = (ctypes.c_void_p(0x10000 * (i + 1)) for i in range(4))
    a.entries, a.tokens = 2, 5
    assert capi.latent_read(_set(a, **over)) == getattr(capi, "ERR_" + want)


@pytest.mark.parametrize("over,want", CACHE_REFUSALS + [
    (dict(rows=-1), "BAD_SHAPE"), (dict(nodes=0), "BAD_SHAPE"), (dict(heads=0), "BAD_SHAPE"), (dict(heads=129), "UNSUPPORTED"),
    (dict(nodes=257), "UNSUPPORTED"), (dict(q=None), "NULL_POINTER"), (dict(out=None), "NULL_POINTER"),
    (dict(q=ctypes.c_void_p(0x10008)), "MISALIGNED"), (dict(out=ctypes.c_void_p(0x20008)), "MISALIGNED"),
    (dict(counts=ctypes.c_void_p(0x20002)), "MISALIGNED"),
    (dict(nodes=33, tree=ctypes.c_void_p(0x70000), tree_words=1), "BAD_SHAPE"),
    (dict(indices=ctypes.c_void_p(0x70000), topk=8, indices_stride=7), "BAD_SHAPE"),
    (dict(indices=ctypes.c_void_p(0x70000), topk=-1), "BAD_SHAPE"),
    (dict(indices=ctypes.c_void_p(0x70000), topk=8, indices_stride=8, nodes=2), "UNSUPPORTED"),
    (dict(indices=ctypes.c_void_p(0x70000), topk=8, indices_stride=8, tree=ctypes.c_void_p(0x70000), tree_words=1), "UNSUPPORTED"),
    (dict(indices=ctypes.c_void_p(0x70000), topk=2 ** 31 - 1, indices_stride=2 ** 31), "UNSUPPORTED"),
    (dict(rows=2 ** 30), "BAD_SHAPE"),
])
def test_latent_decode_refuses_bad_arguments_before_the_device(over, want):
    from qsa_b200 import capi

    a = capi.LatentDecodeArgs()
    a.cache = _cache()
    a.q, a.out = ctypes.c_void_p(0x10000), ctypes.c_void_p(0x20000)
    a.rows, a.nodes, a.heads, a.softmax_scale = 2, 1, 16, 0.07
    a = _set(a, **over)
    assert capi.latent_decode(a) == getattr(capi, "ERR_" + want)
    assert capi.latent_decode_workspace_bytes(a) == getattr(capi, "ERR_" + want)


@pytest.mark.parametrize("over,want", [
    (dict(entries=-1), "BAD_SHAPE"), (dict(heads=0), "BAD_SHAPE"), (dict(q_stride=191), "BAD_SHAPE"),
    (dict(k_stride=127), "BAD_SHAPE"), (dict(v_head_stride=120), "BAD_SHAPE"), (dict(k_rope_stride=63), "BAD_SHAPE"),
    (dict(dtype=2), "UNSUPPORTED"), (dict(q=None), "NULL_POINTER"), (dict(cu_k=None), "NULL_POINTER"),
    (dict(v=None), "NULL_POINTER"), (dict(k=ctypes.c_void_p(0x20008)), "MISALIGNED"), (dict(q_head_stride=196), "MISALIGNED"),
    (dict(k_rope_stride=68), "MISALIGNED"), (dict(cu_q=ctypes.c_void_p(0x60001)), "MISALIGNED"),
])
def test_latent_prefill_refuses_bad_arguments_before_the_device(over, want):
    from qsa_b200 import capi

    a = capi.LatentPrefillArgs()
    a.q, a.k, a.k_rope, a.v, a.out, a.cu_q, a.cu_k = (ctypes.c_void_p(0x10000 * (i + 1)) for i in range(7))
    a.entries, a.q_tokens, a.k_tokens, a.heads, a.softmax_scale = 1, 9, 9, 4, 0.07
    a.q_stride, a.q_head_stride, a.k_stride, a.k_head_stride = 768, 192, 1024, 256
    a.v_stride, a.v_head_stride, a.k_rope_stride = 1024, 256, 64
    assert capi.latent_prefill(_set(a, **over)) == getattr(capi, "ERR_" + want)


def test_empty_calls_need_no_tensors_and_no_device():
    from qsa_b200 import capi

    none = dict(codes=None, rope=None, scales=None, btable=None)
    a = _append_args(tokens=0, c=None, r=None, starts=None, **none)
    assert capi.latent_append(a) == capi.OK
    d = capi.LatentDecodeArgs()
    d.cache = _cache()
    d.nodes, d.heads = 1, 16
    assert capi.latent_decode(_set(d, **none)) == capi.OK and capi.latent_decode_workspace_bytes(d) == 0


def test_latent_cache_refuses_other_ranks():
    from qsa_b200 import latent_cache

    with pytest.raises(ValueError, match="rank"):
        latent_cache(4, 16, 500, device="cpu")
    codes, rope, scales = latent_cache(4, 16, 256, device="cpu")
    assert codes.shape == (4, 16, 256) and rope.shape == (4, 16, 64) and scales.shape == (4, 16)


# ---------------------------------------------------------------- inputs ----
def _gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def _filled(gen, pages, page, rank, spread=1.0):
    """A cache of tokens whose scales are spread over powers of two."""
    codes = (torch.randn((pages, page, rank), generator=gen, device="cuda") * 110).clamp(-448, 448).to(torch.float8_e4m3fn)
    e = (torch.randn((pages, page), generator=gen, device="cuda") * spread).round() - 7
    scales = torch.exp2(e)
    rope = (torch.randn((pages, page, 64), generator=gen, device="cuda") / scales[..., None]).to(torch.bfloat16)
    return codes, rope, scales


def _pages(gen, reqs, per_req, spare=2):
    pool = reqs * per_req + spare
    return torch.randperm(pool, generator=gen, device="cuda")[:reqs * per_req].to(torch.int32).view(reqs, per_req), pool


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------- append ----
def _check_append(before, after, c, r, weight, eps, table, positions, interleaved, place):
    """Cache tensors before and after against the oracle."""
    named, pos, slot = place
    codes0, rope0, scales0 = (t.clone() for t in before)
    rank = codes0.shape[-1]
    live = slot >= 0
    y = L.norm(c, weight, eps)[live]
    rot, size = L.rotate(r, table, pos if positions is None else positions, interleaved)
    rot, size = rot[live], size[live]
    at = slot[live]
    y_err = 16 * U if weight is not None else 0.0
    finite = np.where(np.isfinite(y), np.abs(y), 0.0)
    top = finite.max(1)
    got_s = np64(after[2]).reshape(-1)[at]
    nan = np.isnan(y).any(1)
    assert np.array_equal(np.isnan(got_s), nan)
    lo, hi = L.exponent(top * (1 - y_err)), L.exponent(top * (1 + y_err))
    with np.errstate(invalid="ignore"):
        e = np.log2(np.where(nan, 1.0, got_s))
    assert ((e == lo) | (e == hi) | nan).all()
    # a token with a NaN: zero codes, the rotated part by the scale of the others
    div = np.where(nan, 2.0 ** hi.astype(np.float64), got_s)[:, None]
    tab = O.e4m3fn_table().astype(np.float64)
    got_c = tab[u8(after[0]).reshape(-1, rank)[at]]
    want = np.where(nan[:, None], 0.0, y / div)
    sat = np.clip(want, -448, 448)
    assert not np.isnan(got_c).any()
    assert (np.abs(got_c - sat) <= L.step(sat) / 2 + y_err * np.abs(sat)).all()
    got_r, want_r = np64(after[1]).reshape(-1, 64)[at], rot / div
    fin = np.isfinite(want_r) & (np.abs(want_r) < 3.38e38)
    err = np.abs(np.where(fin, got_r, 0) - np.where(fin, want_r, 0))
    assert (err <= 2.0 ** -8 * np.abs(np.where(fin, want_r, 0)) + 4 * U * np.where(fin, size / div, 0) + 2.0 ** -133).all()
    # all other places stay as they were
    others = np.ones(codes0.shape[0] * codes0.shape[1], bool)
    others[at] = False
    for a, b in zip(before, after):
        w = a.element_size() * a[0, 0].numel()
        x, z = (t.contiguous().view(torch.uint8).view(-1, w).cpu().numpy() for t in (a, b))
        assert np.array_equal(x[others], z[others])


APPEND_CASES = {
    # name: rank, page, lengths, starts, reqs, rotary, interleaved, own positions, norm
    "step": (512, 16, None, [0, 15, 16, 63, 5], None, 64, False, True, True),
    "ragged": (512, 16, [0, 1, 17, 0, 40, 3, 0], [9, 0, 31, 2, 1, 63, 7], [6, 0, 1, 2, 5, 3, 4], 64, True, False, True),
    "plain": (256, 24, [5, 30], [0, 11], None, 0, False, True, False),
    "partial": (384, 7, [9, 2, 1], [3, 0, 40], None, 32, False, False, True),
    "narrow": (128, 1, [4, 4], [0, 2], None, 16, True, True, True),
    "one": (512, 64, [1], [63], None, 64, False, True, False),
    "many": (128, 16, [i % 3 for i in range(1100)], [i % 20 for i in range(1100)], None, 64, False, True, True),
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", sorted(APPEND_CASES))
def test_latent_append_matches_the_oracle(name, dtype):
    import qsa_b200 as qsa

    rank, page, lengths, starts, reqs, rotary, interleaved, own, norm = APPEND_CASES[name]
    gen = _gen(3)
    n = len(starts)
    cu = None if lengths is None else np.concatenate([[0], np.cumsum(lengths)])
    tokens = n if cu is None else int(cu[-1])
    per_req = -(-(max(starts) + max(lengths or [1])) // page)
    btable, pool = _pages(gen, n, per_req)
    before = _filled(gen, pool, page, rank)
    after = tuple(t.clone() for t in before)
    packed = (torch.randn((tokens, rank + 64 + 16), generator=gen, device="cuda") * 3).to(dtype)
    c, r = packed[:, :rank], packed[:, rank:rank + 64]
    weight = (1 + 0.2 * torch.randn(rank, generator=gen, device="cuda")).to(dtype) if norm else None
    table = qsa.rope_table(80, rotary) if rotary else None
    positions = torch.randint(-2, 83, (tokens,), generator=gen, device="cuda", dtype=torch.int32) if rotary and not own else None
    got = qsa.qsa_latent_append(c, r, *after, btable, i32(starts), reqs=None if reqs is None else i32(reqs),
                                cu_tokens=None if cu is None else i32(cu), table=table, positions=positions,
                                c_weight=weight, eps=1e-5, interleaved=interleaved)
    assert all(a is b for a, b in zip(got, after))
    place = L.places(btable.cpu().numpy(), starts, reqs, cu, tokens, page, pool)
    _check_append(before, after, np64(c), np64(r), None if weight is None else np64(weight), 1e-5,
                  None if table is None else np64(table), None if positions is None else positions.cpu().numpy(),
                  interleaved, place)


@pytest.mark.gpu
def test_latent_append_skips_what_lies_outside():
    import qsa_b200 as qsa

    gen = _gen(4)
    before = _filled(gen, 6, 4, 128)
    after = tuple(t.clone() for t in before)
    btable = i32([[0, 9], [1, -1], [2, 3], [4, 5]])
    starts, reqs = [2, 1, -1, 7, 0, 2147483647, 5], [0, 1, 2, 3, -1, 3, 4]
    cu = [1, 5, 9, 11, 14, 15, 17, 18]  # the first token belongs to no entry, nor does the last
    tokens = 19
    c = torch.randn((tokens, 128), generator=gen, device="cuda")
    r = torch.randn((tokens, 64), generator=gen, device="cuda")
    qsa.qsa_latent_append(c, r, *after, btable, i32(starts), reqs=i32(reqs), cu_tokens=i32(cu))
    place = L.places(btable.cpu().numpy(), starts, reqs, cu, tokens, 4, 6)
    _check_append(before, after, np64(c), np64(r), None, 1e-6, None, None, False, place)
    assert (place[2] >= 0).sum() == 2 + 3 + 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rank", RANKS)
def test_latent_append_values_at_the_edges(rank, dtype):
    import qsa_b200 as qsa

    big = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).smallest_normal
    rows = []
    for special in [(0.0,), (448.0,), (1.75 * 2.0 ** 4, -1.0), (1.7578125 * 2.0 ** 4, 1.0), (big, -1.0), (tiny, 0.0),
                    (float("inf"), 3.0), (float("-inf"),), (float("nan"), 2.0), (float("inf"), float("nan")), (448.0, 464.0, 0.0)]:
        row = torch.zeros(rank)
        row[torch.arange(len(special)) * 37 % rank] = torch.tensor(special)
        rows.append(row)
    c = torch.stack(rows).to(dtype).cuda()
    r = torch.randn((len(rows), 64), generator=_gen(1), device="cuda").to(dtype)
    r[0, :3] = torch.tensor([float("inf"), float("nan"), 0.0])
    before = _filled(_gen(2), 3, 8, rank)
    after = tuple(t.clone() for t in before)
    btable = i32([[2, 0]])
    qsa.qsa_latent_append(c, r, *after, btable, i32([3]), cu_tokens=i32([0, len(rows)]))
    place = L.places(btable.cpu().numpy(), [3], None, [0, len(rows)], len(rows), 8, 3)
    _check_append(before, after, np64(c), np64(r), None, 1e-6, None, None, False, place)
    got_r = np64(after[1]).reshape(-1, 64)[place[2][0]]
    assert got_r[0] == np.inf and np.isnan(got_r[1]) and got_r[2] == 0.0


# ------------------------------------------------------------------ read ----
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rank", RANKS)
def test_latent_read_gives_what_the_cache_holds(rank, dtype):
    import qsa_b200 as qsa

    gen = _gen(5)
    codes, rope, scales = _filled(gen, 9, 5, rank, spread=2.0)
    scales.view(-1)[7], scales.view(-1)[8], scales.view(-1)[11] = float("nan"), 0.0, 0.3
    btable = i32([[8, 1, 2], [0, 77, 4], [5, 6, -3]])
    starts, reqs, cu = [2, 0, 14, -1, 0], [2, 1, 0, 0, 5], [0, 9, 24, 27, 29, 31]
    tokens = 34
    c, r = (torch.full((tokens, n), 5.0, dtype=dtype, device="cuda") for n in (rank, 64))
    got = qsa.qsa_latent_read(codes, rope, scales, btable, i32(starts), i32(cu), tokens, reqs=i32(reqs), out=(c, r))
    assert got[0] is c and got[1] is r
    fresh = qsa.qsa_latent_read(codes, rope, scales, btable, i32(starts), i32(cu), tokens, reqs=i32(reqs), dtype=dtype)
    lat, rot = L.values(u8(codes), np64(rope), np64(scales))
    named, pos, slot = L.places(btable.cpu().numpy(), starts, reqs, cu, tokens, 5, 9)
    rel, least = ROUND[dtype]
    for x, y, all_of in ((c, fresh[0], lat), (r, fresh[1], rot)):
        want = np.where((slot >= 0)[:, None], all_of[slot], 0.0)
        a = np64(x)
        assert (a[~named] == 5.0).all() and named.sum() == 31
        a, want, b = a[named], want[named], np64(y)[named]
        assert np.array_equal(np.isnan(a), np.isnan(want)) and np.array_equal(a, b, equal_nan=True)
        fin = ~np.isnan(want) & (np.abs(want) < float(torch.finfo(dtype).max))
        assert (np.abs(a[fin] - want[fin]) <= rel * np.abs(want[fin]) + least).all()


@pytest.mark.gpu
def test_latent_read_one_token_an_entry_and_nothing():
    import qsa_b200 as qsa

    codes, rope, scales = _filled(_gen(6), 4, 3, 256)
    btable = i32([[3, 0], [1, 2]])
    c, r = qsa.qsa_latent_read(codes, rope, scales, btable, i32([4, 2]), None, 2, dtype=torch.float32)
    lat, rot = L.values(u8(codes), np64(rope), np64(scales))
    assert np.array_equal(np64(c), lat[[0 * 3 + 1, 1 * 3 + 2]]) and np.array_equal(np64(r), rot[[1, 5]])
    c, r = qsa.qsa_latent_read(codes, rope, scales, btable, i32([4, 2]), i32([0, 0, 0]), 0)
    assert c.shape == (0, 256) and r.shape == (0, 64) and c.dtype == torch.bfloat16


# ---------------------------------------------------------------- decode ----
def _check_decode(out, q, cache, btable, t2r=None, indices=None, counts=None, tree=None, scale=0.07):
    n4 = q if q.dim() == 4 else q[:, None]
    host = lambda t: None if t is None else t.cpu().numpy()
    want = L.decode(np64(n4), u8(cache[0]), np64(cache[1]), np64(cache[2]), host(btable), host(t2r), host(indices),
                    host(counts), host(tree), scale)
    got = np64(out if out.dim() == 4 else out[:, None])
    assert out.dtype == torch.bfloat16 and out.shape[:-1] == q.shape[:-1]
    for r, w in enumerate(want):
        if w is None:
            assert not got[r].any()
            continue
        assert np.array_equal(np.isnan(got[r]), np.isnan(w["out"])), r
        bound = (2.0 ** -13 * w["score"][..., None] + 2.0 ** -7) * w["size"] + 2.0 ** -16 * w["low"] + 2.0 ** -8 * np.abs(w["out"])
        bad = ~(np.abs(got[r] - w["out"]) <= bound + 2.0 ** -133) & ~np.isnan(w["out"])
        assert not bad.any(), (r, np.argwhere(bad)[:4].tolist(), np.abs(got[r] - w["out"])[bad][:4], bound[bad][:4])


def _queries(gen, rows, nodes, heads, rank, size=1.0):
    q = torch.randn((rows, nodes, heads, rank + 64), generator=gen, device="cuda") * size
    return (q if nodes > 1 else q[:, 0]).to(torch.bfloat16).contiguous()


@pytest.mark.gpu
@pytest.mark.parametrize("rank", RANKS)
@pytest.mark.parametrize("heads", [1, 3, 16, 20, 64, 65, 128])
def test_latent_decode_heads_and_ragged_rows(heads, rank):
    import qsa_b200 as qsa

    gen = _gen(7)
    counts = [0, 1, 2, 63, 64, 65, 127, 128, 129, 300, 511, -1]
    btable, pool = _pages(gen, len(counts), 32)
    cache = _filled(gen, pool, 16, rank)
    q = _queries(gen, len(counts), 1, heads, rank, 0.4)
    out = qsa.qsa_latent_decode(q, *cache, btable, counts=i32(counts), softmax_scale=0.07)
    _check_decode(out, q, cache, btable, counts=i32(counts))


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 3, 16, 24, 64, 100, 128, 256])
@pytest.mark.parametrize("rows,longest", [(1, 1), (2, 33), (3, 2500), (40, 700)])
def test_latent_decode_pages_and_lengths(page, rows, longest):
    import qsa_b200 as qsa

    gen = _gen(8)
    btable, pool = _pages(gen, rows, -(-longest // page))
    cache = _filled(gen, pool, page, 256)
    q = _queries(gen, rows, 1, 5, 256, 0.5)
    counts = torch.randint(0, longest + 1, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    counts[0] = longest
    t2r = torch.randperm(rows, generator=gen, device="cuda").to(torch.int32)
    out = qsa.qsa_latent_decode(q, *cache, btable, t2r, counts=counts, softmax_scale=0.07)
    _check_decode(out, q, cache, btable, t2r, counts=counts)


@pytest.mark.gpu
@pytest.mark.parametrize("columns", [1, 60, 128, 700, 2100])
@pytest.mark.parametrize("rows,heads", [(1, 8), (7, 128), (200, 3)])
def test_latent_decode_selections(rows, heads, columns):
    import qsa_b200 as qsa

    gen = _gen(9)
    reqs, per_req, page = 3, 20, 16
    btable, pool = _pages(gen, reqs, per_req)
    btable[1, 3], btable[2, 0] = -1, pool
    cache = _filled(gen, pool, page, 512)
    q = _queries(gen, rows, 1, heads, 512, 0.3)
    # repeated, unordered, negative and far selections, rows of other tables
    indices = torch.randint(-40, per_req * page + 9, (rows, columns), generator=gen, device="cuda", dtype=torch.int32)
    indices[0, :] = -1 if rows > 1 else indices[0, :]
    t2r = torch.randint(-1, reqs + 1, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    counts = torch.randint(0, columns + 5, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    for c in (None, counts):
        out = qsa.qsa_latent_decode(q, *cache, btable, t2r, indices, counts=c, softmax_scale=0.07)
        _check_decode(out, q, cache, btable, t2r, indices, c)
    wide = torch.full((rows, columns + 7), 1, dtype=torch.int32, device="cuda")
    wide[:, :columns] = indices
    again = qsa.qsa_latent_decode(q, *cache, btable, t2r, wide[:, :columns], counts=counts, softmax_scale=0.07)
    assert torch.equal(again, out)


def _tree(gen, rows, nodes):
    words = -(-nodes // 32)
    bits = np.zeros((rows, nodes, words * 32), bool)
    rng = np.random.default_rng(int(torch.randint(0, 1 << 30, (1,), generator=gen, device="cuda")))
    for e in range(rows):
        for i in range(nodes):
            if i:
                bits[e, i] = bits[e, rng.integers(0, i)]
            bits[e, i, i] = True
    v = (bits.reshape(rows, nodes, words, 32).astype(np.int64) << np.arange(32)).sum(-1)
    return torch.from_numpy(np.where(v >= 1 << 31, v - (1 << 32), v).astype(np.int32)).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("nodes,heads", [(2, 1), (5, 16), (24, 16), (33, 3), (64, 8), (7, 128), (256, 2)])
@pytest.mark.parametrize("kind", ["tree", "chain", "empty bits"])
def test_latent_decode_drafted_nodes(nodes, heads, kind):
    import qsa_b200 as qsa

    gen = _gen(10)
    counts = [nodes, nodes + 1, nodes + 127, 128 + nodes // 2, 600, max(nodes - 1, 0), 0]
    btable, pool = _pages(gen, len(counts), 40)
    cache = _filled(gen, pool, 16, 128)
    q = _queries(gen, len(counts), nodes, heads, 128, 0.5)
    tree = None
    if kind == "tree":
        tree = _tree(gen, len(counts), nodes)
    elif kind == "empty bits":  # a node that sees only the context, one that sees itself, none before them
        tree = torch.zeros((len(counts), nodes, -(-nodes // 32) + 1), dtype=torch.int32, device="cuda")
        tree[:, 1, 0] = 2
        tree[:, :, -1] = -1  # words past the nodes' say nothing
    out = qsa.qsa_latent_decode(q, *cache, btable, counts=i32(counts), tree=tree, softmax_scale=0.07)
    _check_decode(out, q, cache, btable, counts=i32(counts), tree=tree)


@pytest.mark.gpu
def test_latent_decode_reads_nothing_that_is_masked():
    import qsa_b200 as qsa

    gen = _gen(11)
    btable, pool = _pages(gen, 3, 20, spare=4)
    codes, rope, scales = _filled(gen, pool, 16, 512)
    # NaN codes, rotated parts and scales everywhere outside the visible places
    lengths = [1, 130, 300]
    seen = np.zeros(pool * 16, bool)
    for r, n in enumerate(lengths):
        seen[L.slots(btable.cpu().numpy(), r, np.arange(n), 16, pool)] = True
    hide = torch.from_numpy(~seen).cuda().view(pool, 16)
    codes.view(torch.uint8)[hide] = 0x7F
    rope[hide] = float("nan")
    scales[hide] = float("inf")
    q = _queries(gen, 3, 1, 20, 512, 0.3)
    out = qsa.qsa_latent_decode(q, codes, rope, scales, btable, counts=i32(lengths), softmax_scale=0.07)
    _check_decode(out, q, (codes, rope, scales), btable, counts=i32(lengths))
    cols = torch.full((3, 301), -1, dtype=torch.int32, device="cuda")
    for r, n in enumerate(lengths):
        cols[r, torch.randperm(301, generator=gen, device="cuda")[:n]] = torch.arange(n, device="cuda", dtype=torch.int32)
    out = qsa.qsa_latent_decode(q, codes, rope, scales, btable, None, cols, softmax_scale=0.07)
    _check_decode(out, q, (codes, rope, scales), btable, indices=cols)


@pytest.mark.gpu
def test_latent_decode_a_nan_token_shows_where_it_is_seen():
    import qsa_b200 as qsa

    gen = _gen(12)
    btable, pool = _pages(gen, 2, 20)
    cache = _filled(gen, pool, 16, 256)
    nodes, heads = 6, 4
    counts = [206, 150]
    # the third drafted token of the first row is a NaN token, as the append stores it; one of the second's context
    at = L.slots(btable.cpu().numpy(), 0, [203], 16, pool)[0]
    bt = L.slots(btable.cpu().numpy(), 1, [10], 16, pool)[0]
    bad = torch.full((2, 256), float("nan"), device="cuda")
    rot = torch.zeros((2, 64), device="cuda")
    flat = [t.view(-1, 1, *t.shape[2:]) for t in cache]
    qsa.qsa_latent_append(bad, rot, flat[0], flat[1], flat[2], i32([[at], [bt]]), i32([0, 0]))
    q = _queries(gen, 2, nodes, heads, 256, 0.3)
    out = qsa.qsa_latent_decode(q, *cache, btable, counts=i32(counts), softmax_scale=0.07)
    assert torch.isnan(out[0, 3:]).all() and not torch.isnan(out[0, :3]).any() and torch.isnan(out[1]).all()
    _check_decode(out, q, cache, btable, counts=i32(counts))


@pytest.mark.gpu
@pytest.mark.parametrize("columns", [300, 4000])
@pytest.mark.parametrize("spread", ["scales", "scores", "queries", "far scales", "tiny"])
def test_latent_decode_wide_ranges(spread, columns):
    import qsa_b200 as qsa

    gen = _gen(13)
    rows, heads, rank = 2, 12, 512
    btable, pool = _pages(gen, rows, -(-columns // 64))
    codes, rope, scales = _filled(gen, pool, 64, rank)
    q = _queries(gen, rows, 1, heads, rank, 0.3)
    if spread == "scales":
        scales = torch.exp2((torch.randn((pool, 64), generator=gen, device="cuda") * 5).round() - 9)
    elif spread == "scores":
        q = (q * 30).to(torch.bfloat16)
    elif spread == "queries":  # heads whose values differ by many powers of two
        q = (q * torch.exp2(torch.randint(-30, 1, q.shape[:2], generator=gen, device="cuda").float())[..., None]).to(torch.bfloat16)
        q[:, 3] = 0.0
    elif spread == "far scales":  # some tokens of very small values that take a share of the weight, zero ones among them
        small = torch.rand((pool, 64), generator=gen, device="cuda") < 0.3
        scales = torch.where(small, 2.0 ** -60, scales)
        codes.view(torch.uint8)[small & (torch.rand((pool, 64), generator=gen, device="cuda") < 0.3)] = 0
    else:
        scales = torch.full_like(scales, 2.0 ** -60)
    rope = (torch.randn(rope.shape, generator=gen, device="cuda") / scales[..., None]).to(torch.bfloat16)
    counts = i32([columns, columns - 77])
    out = qsa.qsa_latent_decode(q, codes, rope, scales, btable, counts=counts, softmax_scale=0.07)
    _check_decode(out, q, (codes, rope, scales), btable, counts=counts)


@pytest.mark.gpu
def test_latent_decode_past_32_bits_of_offset():
    import qsa_b200 as qsa

    gen = _gen(14)
    page, rank = 4096, 512
    pages = (1 << 33) // (page * rank) + 2  # codes of more than 8 GiB
    codes = torch.zeros((pages, page, rank), dtype=torch.uint8, device="cuda")
    rope = torch.zeros((pages, page, 64), dtype=torch.bfloat16, device="cuda")
    scales = torch.zeros((pages, page), device="cuda")
    part = _filled(gen, 2, page, rank)
    for at, src in ((pages - 1, 0), (0, 1)):
        codes[at], rope[at], scales[at] = part[0].view(torch.uint8)[src], part[1][src], part[2][src]
    btable = i32([[pages - 1, 0]])
    q = _queries(gen, 1, 1, 16, rank, 0.3)
    out = qsa.qsa_latent_decode(q, codes, rope, scales, btable, counts=i32([page + 50]), softmax_scale=0.07)
    _check_decode(out, q, part, i32([[0, 1]]), counts=i32([page + 50]))
    c, r = qsa.qsa_latent_read(codes, rope, scales, btable, i32([0]), i32([0, 100]), 100)
    assert torch.equal(c, part[0][0, :100].to(torch.bfloat16) * part[2][0, :100, None].to(torch.bfloat16))
    x = torch.randn((3, rank), generator=gen, device="cuda")
    qsa.qsa_latent_append(x, x[:, :64], codes, rope, scales, btable, i32([page - 2]), cu_tokens=i32([0, 3]))
    c, _ = qsa.qsa_latent_read(codes, rope, scales, btable, i32([page - 2]), i32([0, 3]), 3, dtype=torch.float32)
    assert (np.abs(np64(c) - np64(x)) <= np.abs(np64(x)).max() / 16).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,columns,heads", [(2, 100, 16), (3, 6000, 16), (2, 3000, 128)])
def test_latent_decode_in_graphs_and_on_a_side_stream(rows, columns, heads):
    import qsa_b200 as qsa

    gen = _gen(15)
    btable, pool = _pages(gen, rows, -(-columns // 16))
    cache = _filled(gen, pool, 16, 512)
    q = _queries(gen, rows, 1, heads, 512, 0.3)
    counts = torch.full((rows,), columns, dtype=torch.int32, device="cuda")
    call = lambda: qsa.qsa_latent_decode(q, *cache, btable, counts=counts, softmax_scale=0.07)
    call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = call()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(call())
    for n in (columns, columns // 3, 0):  # lengths change between replays
        counts.fill_(n)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o in outs:
            _check_decode(o, q, cache, btable, counts=counts)
        if n == columns:
            assert torch.equal(outs[0], eager)
    # calls after one another share nothing: two at once give what one gives
    counts.fill_(columns)
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.current_stream())
        a = [call() for _ in range(4)]
    b = [call() for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, eager) for x in a + b)


# --------------------------------------------------------------- prefill ----
def _check_prefill(out, q, k, k_rope, v, cu_q, cu_k, causal, scale, before=None):
    want, size, score, named = L.prefill(np64(q), np64(k), np64(k_rope), np64(v), cu_q, cu_k, causal, scale)
    got = np64(out)
    rel, least = ROUND[out.dtype]
    bound = (2.0 ** -15 * score[..., None] + 2 * rel + 2.0 ** -12) * size + rel * np.abs(want) + least
    bad = (~(np.abs(got - want) <= bound))[named]
    assert not bad.any(), (np.argwhere(bad)[:4].tolist(), np.abs(got - want)[named][bad][:4], bound[named][bad][:4])
    if before is not None:
        assert np.array_equal(got[~named], np64(before)[~named])


def _prompt(gen, tokens, keys, heads, dtype):
    q = (1.5 * torch.randn((tokens, heads, 192), generator=gen, device="cuda")).to(dtype)
    kv = torch.randn((keys, heads, 256), generator=gen, device="cuda").to(dtype)
    return q, kv[..., :128], torch.randn((keys, 64), generator=gen, device="cuda").to(dtype), kv[..., 128:]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,cached", [
    ([1], [0]), ([0, 1, 2], [0, 0, 0]), ([63, 64, 65], [0, 0, 0]), ([127, 128, 129], [0, 1, 2]),
    ([255, 0, 256, 257], [0, 50, 0, 300]), ([700, 3], [0, 900]), ([10, 200], [-9, -150]), ([5, 4], [-5, -4]), ([1100], [0]),
])
def test_latent_prefill_lengths(lens, cached, causal, dtype):
    import qsa_b200 as qsa

    gen = _gen(20)
    heads = 3
    cu_q = np.concatenate([[0], np.cumsum(lens)])
    cu_k = np.concatenate([[0], np.cumsum(np.array(lens) + cached)])
    q, k, k_rope, v = _prompt(gen, int(cu_q[-1]), int(cu_k[-1]), heads, dtype)
    out = qsa.qsa_latent_prefill(q, k, k_rope, v, i32(cu_q), i32(cu_k), causal=causal, softmax_scale=0.08)
    _check_prefill(out, q, k, k_rope, v, cu_q, cu_k, causal, 0.08)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [1, 2, 16])
def test_latent_prefill_strides_gaps_and_rows_behind(heads):
    import qsa_b200 as qsa

    gen = _gen(21)
    cu_q, cu_k = [3, 140, 140, 300], [7, 150, 160, 500]
    tokens, keys = 320, 530
    q = (1.5 * torch.randn((heads, tokens, 200), generator=gen, device="cuda")).to(torch.bfloat16).permute(1, 0, 2)[..., 8:]
    k = torch.randn((heads, keys, 136), generator=gen, device="cuda").to(torch.bfloat16).permute(1, 0, 2)[..., :128]
    v = torch.randn((keys, heads, 160), generator=gen, device="cuda").to(torch.bfloat16)[..., 32:]
    k_rope = torch.randn((keys, 80), generator=gen, device="cuda").to(torch.bfloat16)[:, 16:]
    # what lies outside the sequences' keys is not read
    for t in (k, v, k_rope):
        t[:7], t[500:] = float("nan"), float("nan")
    out = torch.full((tokens, heads, 128), 9.0, dtype=torch.bfloat16, device="cuda")
    before = out.clone()
    got = qsa.qsa_latent_prefill(q, k, k_rope, v, i32(cu_q), i32(cu_k), out=out)
    assert got is out
    clean = [torch.nan_to_num(t) for t in (k, k_rope, v)]
    _check_prefill(out, q, *clean, cu_q, cu_k, True, 192 ** -0.5, before)


@pytest.mark.gpu
def test_latent_prefill_large_scores_and_no_keys():
    import qsa_b200 as qsa

    gen = _gen(22)
    q, k, k_rope, v = _prompt(gen, 300, 300, 2, torch.bfloat16)
    q = q * 40
    out = qsa.qsa_latent_prefill(q, k, k_rope, v, i32([0, 300]))
    _check_prefill(out, q, k, k_rope, v, [0, 300], [0, 300], True, 192 ** -0.5)
    out = qsa.qsa_latent_prefill(q, k[:0], k_rope[:0], v[:0], i32([0, 300]), i32([0, 0]))
    assert not out.any()
    # a NaN key shows in the queries that see it, and in no other
    k2 = k.clone()
    k2[150, 1, 5] = float("nan")
    out = qsa.qsa_latent_prefill(q, k2, k_rope, v, i32([0, 300]))
    assert torch.isnan(out[150:, 1]).all() and not torch.isnan(out[:150]).any() and not torch.isnan(out[:, 0]).any()


@pytest.mark.gpu
def test_latent_prefill_infinite_and_nan_values_behind_the_mask():
    import qsa_b200 as qsa

    gen = _gen(23)
    q, k, k_rope, v = _prompt(gen, 200, 200, 2, torch.bfloat16)
    v2, r2 = v.clone(), k_rope.clone()
    v2[140:] = float("inf")
    r2[170] = float("nan")
    out = qsa.qsa_latent_prefill(q, k, r2, v2, i32([0, 200]))
    ref = qsa.qsa_latent_prefill(q[:140].contiguous(), k[:140], k_rope[:140], v[:140], i32([0, 140]))
    assert torch.equal(out[:140], ref)


@pytest.mark.gpu
def test_latent_prefill_in_a_graph():
    import qsa_b200 as qsa

    gen = _gen(24)
    q, k, k_rope, v = _prompt(gen, 500, 600, 4, torch.float16)
    cu_q, cu_k = i32([0, 200, 500]), i32([0, 250, 600])
    call = lambda: qsa.qsa_latent_prefill(q, k, k_rope, v, cu_q, cu_k)
    eager = call()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager)
    cu_q.copy_(i32([0, 500, 500]))
    cu_k.copy_(i32([0, 600, 600]))
    g.replay()
    torch.cuda.synchronize()
    _check_prefill(out, q, k, k_rope, v, [0, 500, 500], [0, 600, 600], True, 192 ** -0.5)


# -------------------------------------------------------------- together ----
@pytest.mark.gpu
@pytest.mark.parametrize("rank", [256, 512])
def test_the_latent_operators_together(rank):
    """A prompt in the expanded form, decode steps and a drafted tree in the
    absorbed form, all over one cache: both forms give the same attention."""
    import qsa_b200 as qsa

    gen = _gen(30)
    heads, page, reqs = 4, 16, 3
    lens = [70, 1, 33]
    table = qsa.rope_table(256, 64)
    codes, rope, scales = cache = qsa.latent_cache(40, page, rank)
    btable, _ = _pages(gen, reqs, 8, spare=16)
    wk = torch.randn((heads, 128, rank), generator=gen, device="cuda") / rank ** 0.5
    wv = torch.randn((heads, 128, rank), generator=gen, device="cuda") / rank ** 0.5
    weight = torch.ones(rank, dtype=torch.bfloat16, device="cuda")
    cu = i32(np.concatenate([[0], np.cumsum(lens)]))
    total = sum(lens)
    new = torch.randn((total, rank + 64), generator=gen, device="cuda").to(torch.bfloat16)
    starts = i32([0] * reqs)
    qsa.qsa_latent_append(new[:, :rank], new[:, rank:], *cache, btable, starts, cu_tokens=cu, table=table, c_weight=weight)

    def expanded(q, lengths, cu_q, causal=True):
        """The expanded form over everything cached."""
        cu_k = i32(np.concatenate([[0], np.cumsum(lengths)]))
        c, r = qsa.qsa_latent_read(*cache, btable, starts, cu_k, sum(lengths), dtype=torch.float16)
        k = torch.einsum("td,hed->the", c.float(), wk).half()
        v = torch.einsum("td,hed->the", c.float(), wv).half()
        return qsa.qsa_latent_prefill(q.half(), k, r, v, cu_q, cu_k, causal=causal)

    def absorbed(q, **kw):
        """The absorbed form: queries into the latent's space, its averages out of it."""
        x = torch.cat([torch.einsum("...he,hed->...hd", q[..., :128].float(), wk), q[..., 128:].float()], -1)
        o = qsa.qsa_latent_decode(x.to(torch.bfloat16).contiguous(), *cache, btable, softmax_scale=192 ** -0.5, **kw)
        return torch.einsum("...hd,hed->...he", o.float(), wv)

    # the last token of each prompt, either way
    q = torch.randn((total, heads, 192), generator=gen, device="cuda").to(torch.bfloat16)
    a = expanded(q, lens, cu).float()
    last = cu[1:].long() - 1
    b = absorbed(q[last], counts=i32(lens))
    assert (a[last] - b).abs().max() < 0.05 * a.abs().max()
    # three drafted tokens each: a root and two children
    nodes, depth = 3, [0, 1, 1]
    drafts = torch.randn((reqs * nodes, rank + 64), generator=gen, device="cuda").to(torch.bfloat16)
    positions = i32([n + d for n in lens for d in depth])
    qsa.qsa_latent_append(drafts[:, :rank], drafts[:, rank:], *cache, btable, i32(lens), cu_tokens=i32([0, 3, 6, 9]),
                          table=table, positions=positions, c_weight=weight)
    q = torch.randn((reqs, nodes, heads, 192), generator=gen, device="cuda").to(torch.bfloat16)
    tree = i32([[[0b001], [0b011], [0b101]]] * reqs)
    longer = [n + nodes for n in lens]
    b = absorbed(q, counts=i32(longer), tree=tree)
    chain = absorbed(q, counts=i32(longer))
    a = expanded(q.flatten(0, 1), longer, i32([0, 3, 6, 9])).view(reqs, nodes, heads, 128).float()
    assert (a - chain).abs().max() < 0.05 * a.abs().max()
    assert (a - b)[:, :2].abs().max() < 0.05 * a.abs().max()
    # the third child is accepted: its row moves behind the root's, which is as if it had been drafted there
    acc = drafts.view(reqs, nodes, -1)[:, [0, 2]].reshape(reqs * 2, -1)
    qsa.qsa_latent_append(acc[:, :rank], acc[:, rank:], *cache, btable, i32(lens), cu_tokens=i32([0, 2, 4, 6]), table=table,
                          c_weight=weight)
    again = absorbed(q[:, 2], counts=i32([n + 2 for n in lens]))
    assert (again - b[:, 2]).abs().max() < 0.02 * b.abs().max()


@pytest.mark.gpu
def test_latent_operators_refuse_what_does_not_fit():
    import qsa_b200 as qsa

    gen = _gen(31)
    cache = _filled(gen, 4, 16, 256)
    btable = i32([[0, 1], [2, 3]])
    q = _queries(gen, 2, 1, 8, 256)
    kw = dict(softmax_scale=0.07)
    for bad, match in [
        (lambda: qsa.qsa_latent_decode(q.half(), *cache, btable, **kw), "bfloat16"),
        (lambda: qsa.qsa_latent_decode(q[..., :256].contiguous(), *cache, btable, **kw), "values a head"),
        (lambda: qsa.qsa_latent_decode(q.transpose(0, 1), *cache, btable, **kw), "contiguous"),
        (lambda: qsa.qsa_latent_decode(q, *cache, btable, i32([0]), **kw), "t2r"),
        (lambda: qsa.qsa_latent_decode(q, *cache, btable[:1], **kw), "2 query rows"),
        (lambda: qsa.qsa_latent_decode(q, *cache, btable.long(), **kw), "btable"),
        (lambda: qsa.qsa_latent_decode(q, *cache, btable, tree=i32([[[1]]]), **kw), "tree"),
        (lambda: qsa.qsa_latent_decode(q[:, None].repeat(1, 2, 1, 1), *cache, btable, None, i32([[0], [1]]), **kw), "unsupported|supported"),
        (lambda: qsa.qsa_latent_decode(q.cpu(), *cache, btable, **kw), "q is on|Could not run|device"),
        (lambda: qsa.qsa_latent_decode(q, cache[0], cache[1].float(), cache[2], btable, **kw), "rope"),
        (lambda: qsa.qsa_latent_decode(q, cache[0], cache[1], cache[2][:2], btable, **kw), "scales"),
        (lambda: qsa.qsa_latent_append(q[0, :, :256], q[0, :, 256:].float(), *cache, btable, i32([0, 0])), "dtype"),
        (lambda: qsa.qsa_latent_append(q[0, :2, :255], q[0, :2, 256:], *cache, btable, i32([0, 0])), "c_new"),
        (lambda: qsa.qsa_latent_append(q[0, :3, :256], q[0, :3, 256:], *cache, btable, i32([0, 0])), "one token"),
        (lambda: qsa.qsa_latent_append(q[0, :2, :256], q[0, :2, 256:], *cache, btable, i32([0, 0]), positions=i32([0, 0])), "table"),
        (lambda: qsa.qsa_latent_read(*cache, btable, i32([0, 0]), None, 3), "one token"),
        (lambda: qsa.qsa_latent_read(*cache, btable, i32([0, 0]), None, 2, dtype=torch.float64), "bfloat16"),
        (lambda: qsa.qsa_latent_read(*cache, btable, i32([0, 0]), None, 2, out=(q[0, :3, :256].contiguous(), q[0, :3, :64])), "rows"),
        (lambda: qsa.qsa_latent_prefill(q[..., :192].float(), q[..., :128].float(), q[:, 0, :64].float(), q[..., :128].float(), i32([0, 2])), "bfloat16"),
        (lambda: qsa.qsa_latent_prefill(q[..., :192], q[..., :128], q[:, 0, :64], q[:, :4, :128], i32([0, 2])), "heads"),
        (lambda: qsa.qsa_latent_prefill(q[..., :192], q[..., 4:132], q[:, 0, :64], q[..., :128], i32([0, 2])), "aligned"),
    ]:
        with pytest.raises((RuntimeError, ValueError, NotImplementedError), match=match):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 40])
def test_latent_c_abi_with_a_callers_workspace(rows):
    import qsa_b200 as qsa
    from qsa_b200 import capi

    gen = _gen(32)
    btable, pool = _pages(gen, rows, 60)
    cache = _filled(gen, pool, 16, 512)
    q = _queries(gen, rows, 1, 16, 512, 0.3)
    out = torch.empty((rows, 16, 512), dtype=torch.bfloat16, device="cuda")
    p = lambda t: ctypes.c_void_p(t.data_ptr())
    a = capi.LatentDecodeArgs()
    a.cache = _cache()
    a.cache.codes, a.cache.rope, a.cache.scales, a.cache.btable = p(cache[0]), p(cache[1]), p(cache[2]), p(btable)
    a.cache.pages_per_req = a.cache.btable_stride = 60
    a.cache.num_reqs, a.cache.num_pages = rows, pool
    a.q, a.out, a.rows, a.nodes, a.heads, a.softmax_scale = p(q), p(out), rows, 1, 16, 0.07
    need = capi.latent_decode_workspace_bytes(a)
    ws = torch.empty(need + 512, dtype=torch.uint8, device="cuda").fill_(0xFF)  # needs no clearing
    stream = torch.cuda.current_stream().cuda_stream
    if need:
        assert capi.latent_decode(a, ws, need - 1, stream) == capi.ERR_WORKSPACE
        assert capi.latent_decode(a, None, need, stream) == capi.ERR_WORKSPACE
        assert capi.latent_decode(a, ws[8:], need, stream) == capi.ERR_MISALIGNED
    tail = ws[need:].clone()
    for _ in range(2):  # the second call on what the first one left
        out.zero_()
        assert capi.latent_decode(a, ws if need else None, need, stream) == capi.OK
        torch.cuda.synchronize()
        _check_decode(out, q, cache, btable)
    assert torch.equal(ws[need:], tail)
    assert torch.equal(out, qsa.qsa_latent_decode(q, *cache, btable, softmax_scale=0.07))


# ------------------------------------------------------------ more of each ----
@pytest.mark.gpu
def test_latent_append_and_read_where_entries_end_inside_a_warps_tokens():
    """Entries of 0 to 3 tokens, many of them, some without any, and tokens before and behind them."""
    import qsa_b200 as qsa

    gen = _gen(40)
    counts = torch.randint(0, 4, (700,), generator=gen, device="cuda")
    counts[:5], counts[100:140] = torch.tensor([0, 0, 1, 0, 3], device="cuda"), 0
    cu = torch.cat([torch.full((1,), 3, device="cuda"), 3 + counts.cumsum(0)]).to(torch.int32)
    tokens = int(cu[-1]) + 2
    reqs = torch.randperm(700, generator=gen, device="cuda").to(torch.int32)
    starts = torch.randint(0, 9, (700,), generator=gen, device="cuda", dtype=torch.int32)
    btable, pool = _pages(gen, 700, 4)
    codes, rope, scales = _filled(gen, pool, 3, 128)
    before = codes.clone(), rope.clone(), scales.clone()
    x = torch.randn((tokens, 192), generator=gen, device="cuda", dtype=torch.float32)
    qsa.qsa_latent_append(x[:, :128].contiguous(), x[:, 128:].contiguous(), codes, rope, scales, btable, starts, reqs=reqs, cu_tokens=cu)
    named, pos, slot = place = L.places(btable.cpu().numpy(), starts.cpu().numpy(), reqs.cpu().numpy(), cu.cpu().numpy(), tokens, 3, pool)
    _check_append(before, (codes, rope, scales), np64(x[:, :128]), np64(x[:, 128:]), None, 1e-6, None, None, False, place)
    c = torch.full((tokens, 128), 7.0, device="cuda")
    r = torch.full((tokens, 64), 7.0, device="cuda")
    qsa.qsa_latent_read(codes, rope, scales, btable, starts, cu, tokens, reqs=reqs, out=(c, r))
    lat, rot = L.values(u8(codes), np64(rope), np64(scales))
    assert named[3:-2].all() and not named[:3].any() and not named[-2:].any() and (slot[named] >= 0).all()
    assert np.array_equal(np64(c)[named], lat.reshape(-1, 128)[slot[named]]) and np.array_equal(np64(r)[named], rot.reshape(-1, 64)[slot[named]])
    assert (c[~torch.from_numpy(named).cuda()] == 7).all() and (r[~torch.from_numpy(named).cuda()] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [16, 40])
def test_latent_decode_many_small_weights_beside_a_large_one(heads):
    """20000 tokens of one value, each 2^-17 of one token's weight: together they are
    13 % of the result. Weights may be rounded to 8 bits, and those that share 32
    places with the large one to steps of 2^-15 of it; none of the others is lost."""
    import qsa_b200 as qsa

    rank, n, sink = 256, 20001, 7777
    gen = _gen(41)
    btable, pool = _pages(gen, 1, -(-n // 64))
    latent = torch.zeros((n, rank), device="cuda")
    latent[:, 0], latent[:, 5] = 0.0, 1.0
    latent[sink, 0], latent[sink, 5] = 1.0, 0.0
    codes, rope, scales = qsa.latent_cache(pool, 64, rank)
    qsa.qsa_latent_append(latent, torch.zeros((n, 64), device="cuda"), codes, rope, scales, btable, i32([0]), cu_tokens=i32([0, n]))
    q = torch.zeros((1, heads, rank + 64), device="cuda")
    q[:, :, 0] = 17.0  # log2 of how far the sink's weight is above the others'
    scale = float(np.log(2.0))
    out = np64(qsa.qsa_latent_decode(q.bfloat16(), codes, rope, scales, btable, counts=i32([n]), softmax_scale=scale))
    others = (n - 1) * 2.0 ** -17
    want = others / (1 + others)
    # 2^-7 for the weights in both sums, 2^-8 for the output, 31 tokens that lose all, of 20000
    assert (np.abs(out[0, :, 5] / want - 1) <= 2.0 ** -7 + 2.0 ** -8 + 31 / 20000 + 2.0 ** -12).all(), out[0, :, 5] / want
    assert (np.abs(out[0, :, 0] * (1 + others) - 1) <= 2.0 ** -7 + 2.0 ** -8 + 2.0 ** -12).all()
    assert not out[0, :, 1:5].any() and not out[0, :, 6:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("rank", RANKS)
@pytest.mark.parametrize("order", ["rising", "falling", "steps"])
def test_latent_decode_scores_that_move_far_from_tile_to_tile(rank, order):
    """References pass by more than 2^60 and more than fp32's exponent range between
    the tiles of a row, which two sets of a kernel take in turn."""
    import qsa_b200 as qsa

    gen = _gen(42)
    n = 64 * 9 + 20
    btable, pool = _pages(gen, 2, -(-n // 16))
    cache = _filled(gen, pool, 16, rank, 0.5)
    codes = cache[0].view(torch.uint8)
    level = torch.arange(n, device="cuda") // 64 if order != "steps" else (torch.arange(n, device="cuda") // 64) % 3 * 3
    if order == "falling":
        level = 9 - level
    for r in range(2):
        at = L.slots(btable.cpu().numpy(), r, np.arange(n), 16, pool)
        at = torch.from_numpy(np.asarray(at)).cuda()
        codes.view(-1, rank)[at, 0] = torch.tensor([0x30 + 2 * i for i in range(10)], device="cuda", dtype=torch.uint8)[level]  # 0.5 to 2.25
        cache[2].view(-1)[at] = 1.0
    q = _queries(gen, 2, 1, 33, rank, 0.2)
    q[..., 0] = 900.0
    out = qsa.qsa_latent_decode(q, *cache, btable, counts=i32([n, n - 64]), softmax_scale=0.3)
    _check_decode(out, q, cache, btable, counts=i32([n, n - 64]), scale=0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["tree", "padded"])
def test_latent_decode_reads_no_drafted_token_that_no_node_sees(kind):
    import qsa_b200 as qsa

    gen = _gen(43)
    rows, nodes, heads, rank = 3, 40, 5, 384
    counts = [100, 40, 260]
    btable, pool = _pages(gen, rows, 20)
    cache = _filled(gen, pool, 16, rank)
    tree = np.zeros((rows, nodes, 2), np.int64)
    for i in range(nodes):
        for j in range(i + 1):
            if j not in (3, 17, 33) and (kind == "tree" or i < 30 and j < 30):
                tree[:, i, j // 32] |= 1 << (j % 32)
    unseen = [3, 17, 33] if kind == "tree" else [3, 17] + list(range(30, 40))
    for r, c in enumerate(counts):
        at = torch.from_numpy(np.asarray(L.slots(btable.cpu().numpy(), r, np.array([c - nodes + j for j in unseen]), 16, pool))).cuda()
        cache[0].view(torch.uint8).view(-1, rank)[at] = 0x7F
        cache[1].view(-1, 64)[at] = float("nan")
        cache[2].view(-1)[at] = float("inf")
    words = torch.from_numpy(tree.astype(np.uint32).view(np.int32)).cuda()
    q = _queries(gen, rows, nodes, heads, rank, 0.3)
    out = qsa.qsa_latent_decode(q, *cache, btable, counts=i32(counts), tree=words, softmax_scale=0.07)
    assert not torch.isnan(out).any()
    _check_decode(out, q, cache, btable, counts=i32(counts), tree=words)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,heads", [(600, 3), (1100, 17), (530, 128)])
def test_latent_decode_more_rows_than_threads_plan(rows, heads):
    """Uneven rows, empty ones among them, shared out over all SMs; the requests' pages
    are few, so rows share them."""
    import qsa_b200 as qsa

    gen = _gen(44)
    btable, pool = _pages(gen, 5, 60)
    cache = _filled(gen, pool, 16, 128)
    counts = torch.randint(0, 70, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    counts[::7] = 0
    counts[rows // 2] = 900  # one long row among short ones
    counts[-1] = 640
    t2r = torch.randint(0, 5, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    t2r[rows - 3] = 5  # past the block table
    q = _queries(gen, rows, 1, heads, 128, 0.4)
    out = qsa.qsa_latent_decode(q, *cache, btable, t2r, counts=counts, softmax_scale=0.07)
    # the oracle takes a sample and the special ones
    at = sorted(set(range(0, rows, 37)) | {rows // 2, rows - 1, rows - 3, 7, 8})
    pick = torch.tensor(at, device="cuda")
    _check_decode(out[pick], q[pick], cache, btable, t2r[pick], counts=counts[pick])
    assert not out[::7][counts[::7] == 0].any()
    again = qsa.qsa_latent_decode(q, *cache, btable, t2r, counts=counts, softmax_scale=0.07)
    assert torch.equal(out, again)


@pytest.mark.gpu
@pytest.mark.parametrize("entries", [32, 33, 390, 1000])
def test_latent_prefill_many_entries(entries):
    """Around the numbers of entries that a warp and a block look through at once."""
    import qsa_b200 as qsa

    gen = _gen(45)
    lens = torch.randint(0, 5, (entries,), generator=gen, device="cuda").tolist()
    lens[entries // 2], lens[-1], lens[0] = 300, 70, 0
    more = torch.randint(0, 40, (entries,), generator=gen, device="cuda").tolist()
    cu_q = np.concatenate([[0], np.cumsum(lens)])
    cu_k = np.concatenate([[0], np.cumsum(np.array(lens) + more)])
    q, k, k_rope, v = _prompt(gen, int(cu_q[-1]), int(cu_k[-1]), 2, torch.bfloat16)
    for causal in (True, False):
        out = qsa.qsa_latent_prefill(q, k, k_rope, v, i32(cu_q), i32(cu_k), causal=causal)
        _check_prefill(out, q, k, k_rope, v, cu_q, cu_k, causal, 192 ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,lens,cached", [(1, [700, 30], [400, 0]), (17, [513, 255, 1], [0, 100, 700]), (90, [600], [0]),
                                               (90, [600, 1100], [-400, -600]), (3, [600], [-400])])
def test_latent_prefill_blocks_of_both_sizes(heads, lens, cached, dtype):
    """Few blocks have 256 queries and share out their tiles of keys, many have 512;
    17 and 90 heads are no multiple of those that follow one another; with fewer keys
    than queries the first queries of a block, or half of it, see none."""
    import qsa_b200 as qsa

    gen = _gen(46)
    cu_q = np.concatenate([[0], np.cumsum(lens)])
    cu_k = np.concatenate([[0], np.cumsum(np.array(lens) + cached)])
    q, k, k_rope, v = _prompt(gen, int(cu_q[-1]), int(cu_k[-1]), heads, dtype)
    out = qsa.qsa_latent_prefill(q, k, k_rope, v, i32(cu_q), i32(cu_k), causal=True)
    _check_prefill(out, q, k, k_rope, v, cu_q, cu_k, True, 192 ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [2, 90])
@pytest.mark.parametrize("sign", [1, -1])
def test_latent_prefill_references_that_move(sign, heads, dtype):
    """Scores that rise and fall by more than 2^15, and more than fp32's exponents, from
    tile to tile; a negative scale turns them round."""
    import qsa_b200 as qsa

    gen = _gen(47)
    n = 128 * 7 + 5
    q, k, k_rope, v = _prompt(gen, n, n, heads, dtype)
    q[..., 0] = 40.0
    level = torch.tensor([0.0, 1.0, 6.0, 2.0, 2.5, 20.0, 3.0, 21.0], device="cuda")[torch.arange(n, device="cuda") // 128]
    k = k.clone()
    k[..., 0] = level[:, None].to(dtype)
    out = qsa.qsa_latent_prefill(q, k, k_rope, v, i32([0, n]), i32([0, n]), causal=True, softmax_scale=sign * 0.3)
    _check_prefill(out, q, k, k_rope, v, [0, n], [0, n], True, sign * 0.3)


@pytest.mark.gpu
def test_latent_prefill_two_streams_at_once():
    import qsa_b200 as qsa

    gen = _gen(48)
    q, k, k_rope, v = _prompt(gen, 1500, 1500, 20, torch.bfloat16)
    cu = i32([0, 400, 1500])
    call = lambda: qsa.qsa_latent_prefill(q, k, k_rope, v, cu, cu)
    eager = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = [call() for _ in range(4)]
    b = [call() for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, eager) for x in a + b)


@pytest.fixture
def _wait_limit():
    from qsa_b200 import capi

    capi.device_error(clear=True)
    yield capi
    capi.testing_set_wait_limit_ns(0)
    capi.device_error(clear=True)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["decode", "decode shared out", "prefill", "prefill of few blocks"])
def test_a_latent_wait_that_runs_out_is_reported_and_the_next_call_is_right(which, _wait_limit):
    import qsa_b200 as qsa

    gen = _gen(49)
    if "decode" in which:
        n = 5000 if "shared" in which else 300
        btable, pool = _pages(gen, 2, -(-n // 16))
        cache = _filled(gen, pool, 16, 512)
        q = _queries(gen, 2, 1, 64, 512, 0.3)
        call = lambda: qsa.qsa_latent_decode(q, *cache, btable, counts=i32([n, n - 1]), softmax_scale=0.07)
    else:
        n, heads = 900, 3 if "few" in which else 90
        q, k, k_rope, v = _prompt(gen, n, n, heads, torch.bfloat16)
        call = lambda: qsa.qsa_latent_prefill(q, k, k_rope, v, i32([0, n]), i32([0, n]))
    want = call()
    _wait_limit.testing_set_wait_limit_ns(1)
    call()
    torch.cuda.synchronize()  # the kernel returned: no hang, no fault
    assert _wait_limit.testing_set_wait_limit_ns(0) == 1
    assert _wait_limit.device_error() == 1
    with pytest.raises(RuntimeError, match="device-side failure"):
        _wait_limit.check_device_error(clear=True)
    assert torch.equal(call(), want)
    torch.cuda.synchronize()
    _wait_limit.check_device_error()


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [128, 512])
@pytest.mark.parametrize("rows,n", [(2, 512), (2, 6000), (400, 1500)])
def test_latent_decode_tokens_of_the_least_scale_whose_scores_rise(rows, n, rank):
    """All scales are 2^-60, and from the second tile on scores lie 2^59.5 above the
    first tile's: a sum of weights over scales, taken against the first tile's largest,
    would pass 2^128. Rows that one block has to itself, rows in pieces, and many rows
    shared out. The first tile's weights are 2^-59.5 of the others: below every bound."""
    import qsa_b200 as qsa

    gen = _gen(60)
    reqs, heads = min(rows, 3), 4
    btable, pool = _pages(gen, reqs, -(-n // 64))
    cache = qsa.latent_cache(pool, 64, rank)
    latent = 2.0 ** -55 * (1 + torch.rand((reqs * n, rank), generator=gen, device="cuda"))
    rotated = torch.zeros((reqs * n, 64), device="cuda")
    rotated[:, 0] = torch.where(torch.arange(n, device="cuda").repeat(reqs) < 64, 0.0, 59.5)
    qsa.qsa_latent_append(latent, rotated, *cache, btable, i32([0] * reqs), cu_tokens=i32([n * i for i in range(reqs + 1)]))
    q = torch.zeros((rows, heads, rank + 64), device="cuda")
    q[:, :, rank] = torch.tensor([1.0, 0.5, 0.984375, 0.0], device="cuda")
    t2r = i32([i % reqs for i in range(rows)])
    scale = float(np.log(2.0))
    out = qsa.qsa_latent_decode(q.bfloat16(), *cache, btable, t2r, counts=i32([n] * rows), softmax_scale=scale)
    assert (cache[2].view(-1)[torch.from_numpy(L.slots(btable.cpu().numpy(), 0, np.arange(n), 64, pool)).cuda()] == 2.0 ** -60).all()
    _check_decode(out[:3], q[:3].bfloat16(), cache, btable, t2r[:3], counts=i32([n] * min(rows, 3)), scale=scale)
    # every row has its request's result, however the work was shared out: each is within
    # the bound above, with values above zero 2^-13 * 41.3 + 2^-7 + 2^-8 of it, twice under 2^-4
    got = np64(out)
    want = got[:reqs][np.arange(rows) % reqs]
    assert (np.abs(got - want) <= 2.0 ** -4 * want).all() and (want > 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("columns", [70, 3000])
@pytest.mark.parametrize("heads", [3, 70])
def test_latent_decode_queries_that_are_not_finite(heads, columns):
    """NaN for a head that sees a token, zeros for one that sees none, and nothing of it
    in the other heads: selections without a token, contexts without a page, trees whose
    node sees nothing."""
    import qsa_b200 as qsa

    gen = _gen(61)
    rows, rank = 4, 256
    btable, pool = _pages(gen, rows, -(-columns // 16))
    cache = _filled(gen, pool, 16, rank)
    q = _queries(gen, rows, 1, heads, rank, 0.3)
    clean = q.clone()
    for r, (h, at, x) in enumerate([(0, 5, "nan"), (heads - 1, rank + 40, "inf"), (1, 0, "-inf"), (2, rank, "nan")]):
        q[r, h, at] = float(x)
    bad = torch.isnan(q - q).any(-1)
    indices = torch.arange(columns, device="cuda", dtype=torch.int32).repeat(rows, 1)
    indices[1] = -1
    indices[2, 1:] = -1
    out = qsa.qsa_latent_decode(q, *cache, btable, None, indices, softmax_scale=0.07)
    seen = torch.tensor([True, False, True, True], device="cuda")
    assert not out[1].any()
    assert torch.equal(torch.isnan(out).any(-1), bad & seen[:, None]) and torch.equal(torch.isnan(out).all(-1), bad & seen[:, None])
    ref = qsa.qsa_latent_decode(clean, *cache, btable, None, indices, softmax_scale=0.07)
    assert torch.equal(out[~bad], ref[~bad])
    gone = btable.clone()
    gone[0] = -1
    out = qsa.qsa_latent_decode(q, *cache, gone, softmax_scale=0.07)
    assert not out[0].any() and torch.equal(torch.isnan(out).all(-1), bad & (torch.arange(rows, device="cuda") > 0)[:, None])
    # two nodes that are all there is: the second one's bits are empty
    nodes = torch.stack([q, q], 1).contiguous()
    tree = torch.tensor([1, 0], dtype=torch.int32, device="cuda").repeat(rows, 1).view(rows, 2, 1).contiguous()
    out = qsa.qsa_latent_decode(nodes, *cache, btable, counts=i32([2] * rows), tree=tree, softmax_scale=0.07)
    assert not out[:, 1].any() and torch.equal(torch.isnan(out[:, 0]).all(-1), bad)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,queries,keys", [(1, 100, 300005), (130, 300, 150005)])
def test_latent_prefill_waits_are_for_a_step_and_not_for_a_block(heads, queries, keys, _wait_limit):
    """A limit of 300 looks (30 us of one thread, 1.2 ms of a warp) is ample for every step
    of a block, and less than a block over so many keys takes: 2 ms. Heads lie one behind
    the other in the same memory."""
    import qsa_b200 as qsa

    gen = _gen(62)
    base = torch.randn((keys + heads, 128), generator=gen, device="cuda").to(torch.bfloat16)
    k = base.as_strided((keys, heads, 128), (128, 128, 1))
    k_rope = torch.randn((keys, 64), generator=gen, device="cuda").to(torch.bfloat16)
    q = torch.randn((queries, heads, 192), generator=gen, device="cuda").to(torch.bfloat16)
    cu_q, cu_k = [0, queries], [0, keys]
    call = lambda: qsa.qsa_latent_prefill(q, k, k_rope, k, i32(cu_q), i32(cu_k))
    want = call()
    _wait_limit.testing_set_wait_limit_ns(300 * 1024)
    out = call()
    torch.cuda.synchronize()
    assert _wait_limit.device_error() == 0
    assert torch.equal(out, want)
    at, rows = sorted({0, heads // 2, heads - 1}), [0, queries // 2, queries - 1]
    for i in rows:  # a query alone, over the keys that it sees
        n = keys - (queries - 1 - i)
        _check_prefill(out[i:i + 1, at], q[i:i + 1, at], k[:n, at], k_rope[:n], k[:n, at], [0, 1], [0, n], True, 192 ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("entries,length", [(6, 1500), (300, 5)])
def test_latent_prefill_gives_the_same_again_and_again(entries, length):
    """Blocks of two CTAs that hand memory to one another, several on each SM in turn:
    every call's bits are the first one's, and those are the formula's."""
    import qsa_b200 as qsa

    gen = _gen(63)
    heads = 24
    cu = [length * i for i in range(entries + 1)]
    q, k, k_rope, v = _prompt(gen, cu[-1], cu[-1], heads, torch.bfloat16)
    call = lambda: qsa.qsa_latent_prefill(q, k, k_rope, v, i32(cu))
    want = call()
    for _ in range(40):
        assert torch.equal(call(), want)
    n = min(length, 300)
    at = [0, 7, heads - 1]
    _check_prefill(want[:n, at], q[:n, at], k[:n, at], k_rope[:n], v[:n, at], [0, n], [0, n], True, 192 ** -0.5)


def test_oracle_steps_of_each_32_columns():
    codes = np.zeros((5, 16, 128), np.uint8)
    codes[..., 0] = 0x38  # 1.0
    scales = np.ones((5, 16))
    rope = np.zeros((5, 16, 64))
    rope[2, 3, 0] = 1.0  # column 35
    q = np.zeros((1, 1, 1, 192))
    q[..., 128] = np.log(3.0)
    w = L.decode(q, codes, rope, scales, np.arange(5)[None], counts=[70])[0]
    total = 69 + 3
    assert np.allclose(w["low32"][0, 0, 0], (32 * 1 + 32 * 3 + 6 * 1) / total) and np.allclose(w["low"][0, 0, 0], 70 * 3 / total)
    assert np.allclose(w["spread"][0, 0], 0.0) and np.allclose(w["out"][0, 0, 0], 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("spread", ["even", "scales", "scores", "far scales", "sink"])
@pytest.mark.parametrize("heads,columns", [(12, 4000), (70, 700)])
def test_latent_decode_loses_no_weight_beside_a_larger_one_of_other_columns(heads, columns, spread):
    """The steps of small weights are those of the largest of their 32 columns, not of the
    row: the bound of `_check_decode` with `low32` for `low`. And errors are no larger in
    the mean square than independent roundings of weights and output to 8 bits make them,
    each with a variance of 2^-16 / 3 at most relative to its value, steps of (2^-16)^2 / 3
    of the 32 columns' largest weight, and 2^-13 of a score's terms, which moves each
    token's weight for itself."""
    import qsa_b200 as qsa

    gen = _gen(64)
    rows, rank = 2, 512
    btable, pool = _pages(gen, rows, -(-columns // 64))
    codes, rope, scales = _filled(gen, pool, 64, rank)
    q = _queries(gen, rows, 1, heads, rank, 0.3)
    if spread == "scales":
        scales = torch.exp2((torch.randn((pool, 64), generator=gen, device="cuda") * 5).round() - 9)
    elif spread == "scores":
        q = (q * 30).to(torch.bfloat16)
    elif spread == "far scales":
        scales = torch.where(torch.rand((pool, 64), generator=gen, device="cuda") < 0.3, 2.0 ** -60, scales)
    rope = (torch.randn(rope.shape, generator=gen, device="cuda") / scales[..., None]).to(torch.bfloat16)
    if spread == "sink":  # one token with 2^14 times the weight of the others
        rope[:] = 0
        at = L.slots(btable.cpu().numpy(), 0, [columns // 2], 64, pool)[0]
        q[..., rank:], q[..., :rank] = 0, q[..., :rank] * 0.25
        q[..., rank] = 16.0
        rope.view(-1, 64)[at, 0] = 14 * np.log(2.0) / 0.07 / 16 / float(scales.view(-1)[at])
    counts = i32([columns, columns - 77])
    out = qsa.qsa_latent_decode(q, codes, rope, scales, btable, counts=counts, softmax_scale=0.07)
    host = [u8(codes), np64(rope), np64(scales), btable.cpu().numpy()]
    want = L.decode(np64(q[:, None]), *host, counts=counts.cpu().numpy(), softmax_scale=0.07)
    for r, w in enumerate(want):
        err = np.abs(np64(out)[r] - w["out"][0])
        score = w["score"][0][..., None]
        bound = (2.0 ** -13 * score + 2.0 ** -7) * w["size"][0] + 2.0 ** -16 * w["low32"][0] + 2.0 ** -8 * np.abs(w["out"][0])
        bad = ~(err <= bound + 2.0 ** -133)
        assert not bad.any(), (r, np.argwhere(bad)[:4].tolist(), err[bad][:4], bound[bad][:4])
        mean = 2.0 ** -16 / 3 * (w["out"][0] ** 2 + w["spread"][0]) + 2.0 ** -32 / 3 * w["steps"][0] + 2.0 ** -26 * score ** 2 * w["spread"][0]
        assert (err ** 2).mean() <= mean.mean()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,queries,keys", [(2, 300, 900), (80, 512, 512)])
def test_latent_prefill_errors_are_those_of_its_roundings(heads, queries, keys, dtype):
    """In the mean too: weights and output, each rounded to the type with a variance of
    a third of the square of half a step, and 2^-15 of a score's terms, which moves each
    weight for itself."""
    import qsa_b200 as qsa

    gen = _gen(65)
    q, k, k_rope, v = _prompt(gen, queries, keys, heads, dtype)
    out = qsa.qsa_latent_prefill(q, k, k_rope, v, i32([0, queries]), i32([0, keys]))
    rel = ROUND[dtype][0]
    for h in (0, heads - 1):
        want, size, score, _ = L.prefill(np64(q[:, [h]]), np64(k[:, [h]]), np64(k_rope), np64(v[:, [h]]), [0, queries], [0, keys], True,
                                         192 ** -0.5)
        key = np.concatenate([np64(k[:, h]), np64(k_rope)], 1)
        s = np64(q[:, h]) @ key.T * 192 ** -0.5
        s = np.where(np.arange(keys)[None] <= np.arange(queries)[:, None] + keys - queries, s, -np.inf)
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        err = np64(out[:, h]) - want[:, 0]
        moved = p ** 2 @ np64(v[:, h]) ** 2
        mean = rel ** 2 / 3 * (want[:, 0] ** 2 + moved) + 2.0 ** -30 * score ** 2 * moved
        assert (err ** 2).mean() <= mean.mean()


def test_device_helpers_have_one_definition():
    """Headers that a source may include together define no helper twice."""
    import re
    from pathlib import Path

    seen = {}
    for path in sorted((Path(__file__).resolve().parents[1] / "qsa-fp8-sm89_b200" / "csrc").glob("*.cuh")):
        for name, params in re.findall(r"__device__ __forceinline__ [\w:<>]+ (\w+)\(([^)]*)\)", path.read_text()):
            types = re.sub(r"\b\w+\s*(?=,|$)", "", params).replace(" ", "")
            assert seen.setdefault((name, types), path.name) == path.name, (name, path.name, seen[name, types])
    assert ("fma2", "uint64_t,uint64_t,uint64_t") in seen
