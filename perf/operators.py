"""Measured cases of the block-scaled cache's operators.

Three operators serve one attention layer over a paged E4M3FN cache that keeps
a scale for each block of tokens and KV head:

* ``qk_rope``: RMS norm of every query and key head and the position rotation,
  one or three position axes, from a packed projection;
* ``append``: new keys (normed and rotated on the way) and values into the
  paged cache, quantised with the scale of their block;
* ``decode``: grouped-query attention over that cache, over Top-K selections
  or over whole contexts, with an optional sigmoid gate.

``run`` computes them in elementary torch operations in 32 bits, or, where
``own`` is true, by the framework's entry points.
"""

import math
import sys
from pathlib import Path

import torch

own = False

D = 128
E4M3_MAX = 448.0
TINY = 2.0 ** -126
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# pairs of each axis (time, height, width) in eighths of the rotated pairs
SECTION_EIGHTHS = (2, 3, 3)


def _package():
    root = str(Path(__file__).resolve().parents[1] / "qsa-fp8-sm89_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import qsa_b200

    return qsa_b200


# ------------------------------------------------------------------ cases ----
def listed():
    rope = dict(op="qk_rope", hq=32, hkv=8, rotary=128, interleaved=False, axes=1, norm=True, dtype="bf16")
    app = dict(op="append", hkv=8, page=16, block=16, rotary=128, interleaved=False, axes=1, norm=True, dtype="bf16")
    dec = dict(op="decode", hq=32, hkv=8, page=16, block=16, per_req=1, gate=True)
    return [
        # one decode step of four requests: the call's latency
        dict(rope, name="rope_step_4", tokens=4),
        # one decode step of a full batch, partial rotation in adjacent pairs
        dict(rope, name="rope_step_256", tokens=256, hq=64, rotary=64, interleaved=True, dtype="f16"),
        # a ragged image prompt in full precision, three position axes
        dict(rope, name="rope_image_1531", tokens=1531, hq=24, hkv=4, axes=3, dtype="f32"),
        # a long prompt's prefill
        dict(rope, name="rope_prefill_16384", tokens=16384),
        # one token of each of 256 requests, inside their blocks and at block starts
        dict(app, name="append_step_256", reqs=256, new_lo=1, new_hi=1, ctx_lo=0, ctx_hi=511),
        # speculative tokens, page and block that are no powers of two, no rotation
        dict(app, name="append_spec_93", reqs=93, new_lo=0, new_hi=7, ctx_lo=1, ctx_hi=3000, hkv=5, page=24, block=12,
             rotary=0, norm=False, dtype="f16"),
        # prompts of uneven length, one scale a page
        dict(app, name="append_prefill_24", reqs=24, new_lo=256, new_hi=4096, ctx_lo=0, ctx_hi=700, page=64, block=64),
        # the smallest configuration: 4 requests, every one of 64 tokens
        dict(dec, name="decode_4x64", rows=4, ctx=64, topk=64, len_lo=64, len_hi=64),
        # the headline configuration: 256 requests, 512 of 512 tokens
        dict(dec, name="decode_256x512", rows=256, ctx=512, topk=512, len_lo=512, len_hi=512),
        # ragged selections from long contexts, several query rows a request
        dict(dec, name="decode_512x2048_ragged", rows=512, per_req=4, hq=64, ctx=16384, topk=2048, len_lo=64,
             len_hi=2048),
        # whole long contexts, few rows: the context is split
        dict(dec, name="decode_dense_8x131072", rows=8, hq=64, ctx=131072, topk=0, len_lo=90001, len_hi=131072, page=64,
             block=64),
        # whole contexts of uneven length, empty ones among them, one KV head, no gate
        dict(dec, name="decode_dense_61_mqa", rows=61, hq=20, hkv=1, ctx=6000, topk=0, len_lo=0, len_hi=6000, page=48,
             block=8, gate=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["qk_rope", "append", "decode", "decode"])
    if op == "qk_rope":
        hkv = rng.choice([1, 2, 4, 5, 8])
        return dict(op=op, tokens=_log(rng, 1, 16384), hq=hkv * rng.choice([1, 2, 3, 4, 8]) if hkv < 8 else rng.choice([8, 32]),
                    hkv=hkv, rotary=rng.choice([32, 64, 128, 128]), interleaved=rng.random() < 0.3,
                    axes=rng.choice([1, 1, 3]), norm=rng.random() < 0.8, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
    page, block = rng.choice([(1, 1), (16, 16), (16, 16), (16, 4), (24, 12), (32, 16), (48, 8), (64, 64), (64, 1), (128, 128)])
    if op == "append":
        hi = _log(rng, 1, 2048)
        lo = hi if hi == 1 else rng.randint(0, hi)
        reqs = max(1, min(512, _log(rng, 1, 512), 49152 // max(1, (lo + hi) // 2)))
        rotary = rng.choice([0, 64, 128, 128])
        return dict(op=op, reqs=reqs, new_lo=lo, new_hi=hi, ctx_lo=0, ctx_hi=min(_log(rng, 1, 4000), 600000 // reqs),
                    hkv=rng.choice([1, 2, 5, 8]),
                    page=page, block=block, rotary=rotary, interleaved=rng.random() < 0.3,
                    axes=rng.choice([1, 1, 3]) if rotary else 1, norm=rng.random() < 0.8,
                    dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
    hkv = rng.choice([1, 2, 3, 4, 8, 8])
    group = rng.choice([1, 2, 4, 4, 5, 7, 8, 8, 12, 16])
    per_req = rng.choice([1, 1, 2, 4])
    dense = rng.random() < 0.5
    # entries of all rows and their bytes stay under those of the largest listed case
    entries = _log(rng, 64, 900000 // max(1, hkv // 8 + hkv // 4))
    rows = _log(rng, 1, min(768, entries))
    length = max(1, entries // rows)
    length = min(length, 100000 if dense else 3000)
    lo = rng.randint(0, length)
    ctx = length if dense else max(length, min(_log(rng, length, 20 * length), 32768, max(length, 1500000 // rows)))
    return dict(op=op, rows=rows, per_req=min(per_req, rows), hq=hkv * group, hkv=hkv, page=page, block=block, ctx=ctx,
                topk=0 if dense else length, len_lo=lo, len_hi=length, gate=rng.random() < 0.7)


# ------------------------------------------------------------------ inputs ----
def _spread(lo, hi, n, gen):
    """n whole numbers from lo to hi, evenly spread, in an order of the seed."""
    x = lo + (torch.arange(n, device="cuda", dtype=torch.float64) * ((hi - lo) / max(1, n - 1))).round()
    return x[torch.randperm(n, generator=gen, device="cuda")].to(torch.int32)


def _spread_sum(lo, hi, n):
    return int(sum(lo + round(i * ((hi - lo) / max(1, n - 1))) for i in range(n)))


def _table(length, rotary):
    """cos, then sin, of every position's rotation angles, from 64 bits."""
    freq = 500000.0 ** (-torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary)
    ang = torch.arange(length, device="cuda", dtype=torch.float64)[:, None] * freq
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def _sections(rotary):
    a, b = (e * rotary // 16 for e in SECTION_EIGHTHS[:2])
    return (a, b, rotary // 2 - a - b)


def _heads(shape, gen, dtype):
    """Projection outputs: normal values with a few large channels, as trained heads have them."""
    x = torch.randn(shape, generator=gen, device="cuda")
    gain = 1.0 + 7.0 * (torch.rand(shape[-1], generator=gen, device="cuda") > 0.98)
    return (x * gain).to(dtype)


def _codes(shape, gen):
    """Stored E4M3FN values whose blocks reach towards 448."""
    out = torch.empty(shape, dtype=torch.uint8, device="cuda")
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 27):
        x = torch.randn(min(1 << 27, flat.numel() - i), generator=gen, device="cuda", dtype=torch.float32)
        flat[i:i + (1 << 27)] = x.mul_(110.0).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
    return out.view(torch.float8_e4m3fn)


def _scales(shape, gen):
    return 0.01 * torch.exp2(torch.rand(shape, generator=gen, device="cuda") * 3 - 1.5)


def _pages(reqs, per_req, gen):
    """A block table over a shuffled pool with a few spare pages."""
    pool = reqs * per_req + 3
    return torch.randperm(pool, generator=gen, device="cuda")[:reqs * per_req].to(torch.int32).view(reqs, per_req), pool


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case)
    if case["op"] == "qk_rope":
        n, hq, hkv, dt = case["tokens"], case["hq"], case["hkv"], DTYPES[case["dtype"]]
        qkv = _heads((n, hq + 2 * hkv, D), gen, dt)
        limit = 32768
        s.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], table=_table(limit, case["rotary"]),
                 positions=torch.randint(0, limit, (n,) if case["axes"] == 1 else (case["axes"], n), generator=gen,
                                         device="cuda", dtype=torch.int32),
                 sections=None if case["axes"] == 1 else _sections(case["rotary"]))
        for w in ("q_weight", "k_weight"):
            s[w] = (1 + 0.2 * torch.randn(D, generator=gen, device="cuda")).to(dt) if case["norm"] else None
    elif case["op"] == "append":
        n, hkv, page, block, dt = case["reqs"], case["hkv"], case["page"], case["block"], DTYPES[case["dtype"]]
        count = _spread(case["new_lo"], case["new_hi"], n, gen)
        starts = _spread(case["ctx_lo"], case["ctx_hi"], n, gen)
        total = _spread_sum(case["new_lo"], case["new_hi"], n)
        limit = case["ctx_hi"] + case["new_hi"] + 1
        btable, pool = _pages(n, -(-limit // page), gen)
        kv = _heads((total, 2 * hkv, D), gen, dt)
        s.update(k_new=kv[:, :hkv], v_new=kv[:, hkv:], starts=starts, btable=btable,
                 k_cache=_codes((pool, page, hkv, D), gen), v_cache=_codes((pool, page, hkv, D), gen),
                 k_scales=_scales((pool, page // block, hkv), gen), v_scales=_scales((pool, page // block, hkv), gen),
                 cu_tokens=None, positions=None, table=None, sections=None, k_weight=None)
        if not case["new_lo"] == case["new_hi"] == 1:
            s["cu_tokens"] = torch.cat([torch.zeros_like(count[:1]), count.cumsum(0, dtype=torch.int32)])
        if case["rotary"]:
            s["table"] = _table(limit, case["rotary"])
        if case["axes"] > 1:
            s["positions"] = torch.randint(0, limit, (case["axes"], total), generator=gen, device="cuda", dtype=torch.int32)
            s["sections"] = _sections(case["rotary"])
        if case["norm"]:
            s["k_weight"] = (1 + 0.2 * torch.randn(D, generator=gen, device="cuda")).to(dt)
    else:
        rows, hq, hkv, page, block, ctx = (case[x] for x in ("rows", "hq", "hkv", "page", "block", "ctx"))
        reqs = -(-rows // case["per_req"])
        btable, pool = _pages(reqs, -(-ctx // page), gen)
        q = torch.randn((rows, hq, D), generator=gen, device="cuda")
        s.update(q=q.to(torch.bfloat16), gate=None, btable=btable,
                 t2r=torch.arange(rows, device="cuda", dtype=torch.int32) // case["per_req"],
                 counts=_spread(case["len_lo"], case["len_hi"], rows, gen), indices=None,
                 k_cache=_codes((pool, page, hkv, D), gen), v_cache=_codes((pool, page, hkv, D), gen),
                 k_scales=_scales((pool, page // block, hkv), gen), v_scales=_scales((pool, page // block, hkv), gen))
        if case["gate"]:
            s["gate"] = torch.randn((rows, hq, D), generator=gen, device="cuda").to(torch.bfloat16)
        if case["topk"]:
            picks = torch.rand((rows, ctx), generator=gen, device="cuda").argsort(1)[:, :case["topk"]].to(torch.int32)
            past = torch.arange(case["topk"], device="cuda")[None, :] >= s["counts"][:, None]
            s["indices"] = picks.masked_fill_(past, -1).contiguous()
            s["counts"] = None
    return s


# ------------------------------------------------------------- plain forms ----
def _norm_rotate(x, weight, table, positions, sections, interleaved):
    """x[tokens, heads, 128] in 32 bits: RMS norm of each head, then the rotation."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    if table is None:
        return x
    rotary = table.shape[1]
    half = rotary // 2
    if sections is None:
        cs = table[positions.long()]
        cos, sin = cs[:, None, :half], cs[:, None, half:]
    else:
        pair = torch.arange(half, device=x.device)[None, :]
        axis = (pair[0] >= sections[0]).long() + (pair[0] >= sections[0] + sections[1]).long()
        at = positions.long().t()[:, axis]
        cos, sin = table[at, pair][:, None], table[at, half + pair][:, None]
    if interleaved:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:rotary]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rotary:]], -1)


def _to_e4m3(x):
    return x.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _plain_append(s):
    page, hkv = s["k_cache"].shape[1:3]
    block = page // s["k_scales"].shape[1]
    n, tokens = s["starts"].shape[0], s["k_new"].shape[0]
    dev = s["k_new"].device
    cu = s["cu_tokens"].long() if s["cu_tokens"] is not None else torch.arange(n + 1, device=dev)
    starts = s["starts"].long()
    token = torch.arange(tokens, device=dev)
    req = torch.searchsorted(cu, token, right=True) - 1
    pos = starts[req] + token - cu[req]
    slot = s["btable"].long()[req, pos // page] * page + pos % page
    held = pos - pos % block < starts[req]  # the token's block keeps earlier tokens
    # the blocks that the requests' first tokens fall in, and their earlier rows
    off = torch.arange(block, device=dev)[None, :]
    base = starts - starts % block
    first = s["btable"].long()[torch.arange(n, device=dev), base // page] * page + base % page
    keep = (off < (starts % block)[:, None]) & (cu[1:] > cu[:-1])[:, None]
    k = _norm_rotate(s["k_new"], s["k_weight"], s["table"], pos if s["positions"] is None else s["positions"],
                     s["sections"], s["case"]["interleaved"])
    for x, cache, scales in ((k, s["k_cache"], s["k_scales"]), (s["v_new"].float(), s["v_cache"], s["v_scales"])):
        flat, rows = scales.view(-1, hkv), cache.view(torch.uint8).view(-1, hkv, D)
        old = flat.clone()
        flat[slot // block] = torch.where(held[:, None], flat[slot // block], torch.zeros_like(flat[:1]))
        flat.index_reduce_(0, slot // block, (x.abs().amax(-1) / E4M3_MAX).clamp_min(TINY), "amax")
        at = first[:, None] + off
        was = rows[at].view(torch.float8_e4m3fn).float()
        ratio = (old[first // block] / flat[first // block])[:, None, :, None]
        again = torch.where(keep[..., None, None], was * ratio, was)
        rows[at] = _to_e4m3(again).view(torch.uint8)
        rows[slot] = _to_e4m3(x / flat[slot // block][..., None]).view(torch.uint8)
    return s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"]


def _plain_decode(s):
    q, kc, vc = s["q"].float(), s["k_cache"], s["v_cache"]
    rows, hq = q.shape[:2]
    page, hkv = kc.shape[1:3]
    block = page // s["k_scales"].shape[1]
    if s["indices"] is None:
        t = torch.arange(s["btable"].shape[1] * page, device=q.device)[None, :].expand(rows, -1)
        ok = t < s["counts"][:, None]
        t = torch.where(ok, t, 0)
    else:
        t = s["indices"].long()
        ok = t >= 0
        t = torch.where(ok, t, 0)
    slot = s["btable"].long()[s["t2r"].long()[:, None], t // page] * page + t % page
    k = kc.view(torch.uint8).view(-1, hkv, D)[slot].view(torch.float8_e4m3fn).float()
    k *= s["k_scales"].view(-1, hkv)[slot // block][..., None]
    score = torch.matmul(q.view(rows, hkv, hq // hkv, D), k.permute(0, 2, 3, 1)) * D ** -0.5
    del k
    score = torch.where(ok[:, None, None, :], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    v = vc.view(torch.uint8).view(-1, hkv, D)[slot].view(torch.float8_e4m3fn).float()
    v *= s["v_scales"].view(-1, hkv)[slot // block][..., None]
    out = torch.matmul(p, v.transpose(1, 2)).reshape(rows, hq, D)
    if s["gate"] is not None:
        out = out / (1 + torch.exp(-s["gate"].float()))
    return out.to(torch.bfloat16)


def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        qsa = _package()
        if op == "qk_rope":
            return qsa.qsa_qk_rope(s["q"], s["k"], s["table"], s["positions"], q_weight=s["q_weight"],
                                   k_weight=s["k_weight"], eps=EPS, interleaved=s["case"]["interleaved"],
                                   sections=s["sections"])
        if op == "append":
            return qsa.qsa_block_append(s["k_new"], s["v_new"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"],
                                        s["btable"], s["starts"], cu_tokens=s["cu_tokens"], table=s["table"],
                                        positions=s["positions"], k_weight=s["k_weight"], eps=EPS,
                                        interleaved=s["case"]["interleaved"], sections=s["sections"])
        return qsa.qsa_block_decode(s["q"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["btable"],
                                    s["t2r"], s["indices"], gate=s["gate"], counts=s["counts"])
    if op == "qk_rope":
        return tuple(_norm_rotate(s[x], s[x + "_weight"], s["table"], s["positions"], s["sections"],
                                  s["case"]["interleaved"]).to(s[x].dtype) for x in ("q", "k"))
    return _plain_append(s) if op == "append" else _plain_decode(s)


# ------------------------------------------------------------------- work ----
def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}.get(case.get("dtype"), 2)
    if case["op"] == "qk_rope":
        values = case["tokens"] * (case["hq"] + case["hkv"]) * D
        return {"bytes": 2 * size * values + case["tokens"] * 4 * (case["rotary"] + case["axes"]), "flops": 8 * values}
    if case["op"] == "append":
        n, block = case["reqs"], case["block"]
        tokens = _spread_sum(case["new_lo"], case["new_hi"], n)
        rows = 2 * tokens * case["hkv"]
        scales = 2 * 4 * case["hkv"] * max(tokens // block, min(tokens, n))
        return {"bytes": rows * D * (size + 1) + scales + tokens * 4 * case["rotary"] + 12 * n, "flops": 8 * rows * D}
    entries = _spread_sum(case["len_lo"], case["len_hi"], case["rows"])
    # a page's block has one scale for each head; rows of one request may name the same tokens, each row reads them
    kv = entries * case["hkv"] * 2 * (D + (4 if case["topk"] else 4 / case["block"]))
    rest = case["rows"] * case["hq"] * D * 2 * (3 if case["gate"] else 2) + (entries * 4 if case["topk"] else 0)
    return {"bytes": kv + rest, "flops": 4.0 * entries * case["hq"] * D}


# ------------------------------------------------------------ in 64 bits ----
def _exact_norm_rotate(x, weight, table, positions, sections, interleaved):
    x = x.double()
    if weight is not None:
        x = x / ((x ** 2).sum(-1, keepdim=True) / D + EPS).sqrt() * weight.double()
    if table is None:
        return x
    half = table.shape[1] // 2
    out = x.clone()
    axis = 0
    for j in range(half):
        if sections is not None:
            axis = 0 if j < sections[0] else 1 if j < sections[0] + sections[1] else 2
        at = positions.long() if sections is None else positions[axis].long()
        z = torch.complex(table[at, j].double(), table[at, half + j].double())[:, None]
        i, k = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
        turned = torch.complex(x[..., i], x[..., k]) * z
        out[..., i], out[..., k] = turned.real, turned.imag
    return out


def _round_e4m3(x):
    """The nearest E4M3FN value, ties to even, saturated, in 64 bits."""
    a = x.abs().clamp_max(E4M3_MAX)
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3)
    return torch.round(a / step) * step * x.sign()


def _exact_append(s):
    page, hkv = s["k_cache"].shape[1:3]
    block = page // s["k_scales"].shape[1]
    n = s["starts"].shape[0]
    cu = s["cu_tokens"].tolist() if s["cu_tokens"] is not None else list(range(n + 1))
    starts, pages = s["starts"].tolist(), s["btable"].tolist()
    pos = torch.cat([torch.arange(a, a + e - b) for a, b, e in zip(starts, cu, cu[1:])] or [torch.zeros(0)]).to(s["k_new"].device)
    k = _exact_norm_rotate(s["k_new"], s["k_weight"], s["table"], pos if s["positions"] is None else s["positions"],
                           s["sections"], s["case"]["interleaved"])
    out = []
    for x, cache, scales in ((k, s["k_cache"], s["k_scales"]), (s["v_new"].double(), s["v_cache"], s["v_scales"])):
        codes, sc = cache.double().view(-1, block, hkv, D), scales.double().view(-1, hkv)
        for r in range(n):
            done, total = 0, cu[r + 1] - cu[r]
            if not total:
                continue
            # whole rows of blocks: what the first block keeps, the new tokens, and what stays behind the last of them
            lead = starts[r] % block
            count = -(-(lead + total) // block)
            ids = torch.tensor([pages[r][p // page] * (page // block) + p % page // block
                                for p in range(starts[r] - lead, starts[r] - lead + count * block, block)], device=x.device)
            grid = torch.zeros((count * block, hkv, D), dtype=torch.float64, device=x.device)
            grid[lead:lead + total] = x[cu[r]:cu[r + 1]]
            grid = grid.view(count, block, hkv, D)
            new = (grid.abs().amax((1, 3)) / E4M3_MAX).clamp_min(TINY)
            old = codes[ids]
            if lead:
                was = sc[ids[0]]
                new[0] = torch.maximum(new[0], was)
                old[0, :lead] = _round_e4m3(old[0, :lead] * (was / new[0])[None, :, None])
            fresh = torch.zeros(count * block, dtype=torch.bool, device=x.device)
            fresh[lead:lead + total] = True
            fresh = fresh.view(count, block)[..., None, None]
            codes[ids] = torch.where(fresh, _round_e4m3(grid / new[:, None, :, None]), old)
            sc[ids] = new
        out.append((codes.view(cache.shape), sc.view(scales.shape)))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_decode(s):
    rows, hq = s["q"].shape[:2]
    page, hkv = s["k_cache"].shape[1:3]
    block = page // s["k_scales"].shape[1]
    kc, vc = (s[x].view(torch.uint8).view(-1, hkv, D) for x in ("k_cache", "v_cache"))
    ks, vs = (s[x].view(-1, hkv).double() for x in ("k_scales", "v_scales"))
    out = torch.zeros((rows, hq, D), dtype=torch.float64, device=s["q"].device)
    counts = s["counts"].tolist() if s["indices"] is None else (s["indices"] >= 0).sum(1).tolist()
    for r in range(rows):
        if not counts[r]:
            continue
        t = torch.arange(counts[r], device=out.device) if s["indices"] is None else s["indices"][r].long()[:counts[r]]
        slot = s["btable"][s["t2r"][r].long()].long()[t // page] * page + t % page
        k = kc[slot].view(torch.float8_e4m3fn).double() * ks[slot // block][..., None]
        v = vc[slot].view(torch.float8_e4m3fn).double() * vs[slot // block][..., None]
        score = torch.einsum("ghd,tgd->ght", s["q"][r].double().view(hkv, -1, D), k) / math.sqrt(D)
        out[r] = torch.einsum("ght,tgd->ghd", torch.softmax(score, -1), v).reshape(hq, D)
    if s["gate"] is not None:
        out *= torch.sigmoid(s["gate"].double())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "qk_rope":
        return tuple(_exact_norm_rotate(s[x], s[x + "_weight"], s["table"], s["positions"], s["sections"],
                                        case["interleaved"]) for x in ("q", "k"))
    return _exact_append(s) if case["op"] == "append" else _exact_decode(s)
