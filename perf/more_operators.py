"""Measured cases of the latent cache's operators.

A token of latent attention is one vector for all heads: ``rank`` latent values
that serve as key and value, and 64 rotated key values. The paged cache holds
E4M3FN codes of the latent, the rotated part in bf16 and one scale a token::

    key   = scale * (codes, rope)        value = scale * codes

* ``append``: RMS norm of new latents, rotation of their rotated part,
  quantising, into the paged cache;
* ``read``: contexts back out of the cache, for the expanded form;
* ``decode``: the absorbed form, queries in the latent's space attend to the
  cache itself: Top-K selections, whole contexts, trees of drafted tokens;
* ``prefill``: the expanded form for prompts, keys of 128 values a head and 64
  shared ones, values of 128.

``run`` computes them in elementary torch operations in 32 bits, or, where
``own`` is true, by the framework's entry points.
"""

import math
import sys
from pathlib import Path

import torch

own = False

ROPE = 64
HEAD = 128
E4M3_MAX = 448.0
EPS = 1e-6
SCALE = (HEAD + ROPE) ** -0.5
# exponents of a token's scale, a power of two
E_LOW, E_HIGH = -60, 60
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _package():
    root = str(Path(__file__).resolve().parents[1] / "qsa-fp8-sm89_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import qsa_b200

    return qsa_b200


# ------------------------------------------------------------------ cases ----
def listed():
    app = dict(op="append", rank=512, page=16, rope=True, interleaved=False, norm=True, dtype="bf16", own_pos=True)
    read = dict(op="read", rank=512, page=16, dtype="bf16")
    dec = dict(op="decode", rank=512, page=16, heads=32, nodes=1, topk=0, tree=False)
    pre = dict(op="prefill", heads=32, causal=True, dtype="bf16", cached_hi=0)
    return [
        # one token of each of 256 requests: a decode step's append
        dict(app, name="latent_append_step_256", reqs=256, new_lo=1, new_hi=1, ctx_lo=0, ctx_hi=511),
        # prompts of uneven length, and drafted tokens' positions given by the caller
        dict(app, name="latent_append_prefill_24", reqs=24, new_lo=255, new_hi=4097, ctx_lo=0, ctx_hi=700, page=64,
             interleaved=True, dtype="f16", own_pos=False),
        # cached prefixes of a few chunked prompts
        dict(read, name="latent_read_3", reqs=3, len_lo=1, len_hi=777, rank=256, page=24, dtype="f32"),
        # whole contexts for the expanded form
        dict(read, name="latent_read_24", reqs=24, len_lo=511, len_hi=8192, page=64),
        # the smallest configuration: 4 requests of 64 tokens
        dict(dec, name="latent_decode_4x64", rows=4, ctx=64, len_lo=64, len_hi=64, heads=16),
        # the headline selection: 256 requests, 512 selected tokens of 8192
        dict(dec, name="latent_decode_256_topk512", rows=256, ctx=8192, topk=512, len_lo=512, len_hi=512),
        # uneven whole contexts, empty ones among them, odd heads and pages
        dict(dec, name="latent_decode_dense_61", rows=61, ctx=6000, len_lo=0, len_hi=6000, heads=20, rank=256, page=48),
        # few long contexts: the context is split
        dict(dec, name="latent_decode_dense_8x131072", rows=8, ctx=131072, len_lo=90001, len_hi=131072, heads=16, page=64),
        # every head of a wide model on one GPU
        dict(dec, name="latent_decode_dense_32_wide", rows=32, ctx=8192, len_lo=4096, len_hi=8192, heads=128, page=64),
        # trees of 24 drafted tokens over contexts
        dict(dec, name="latent_tree_16x24", rows=16, nodes=24, tree=True, ctx=8192, len_lo=700, len_hi=8192, heads=16),
        # a chunk of a prompt behind cached tokens, and a few short ones
        dict(pre, name="latent_prefill_chunks_5", reqs=5, len_lo=1, len_hi=700, heads=16, cached_hi=2000, dtype="f16"),
        # prompts of uneven length
        dict(pre, name="latent_prefill_6", reqs=6, len_lo=513, len_hi=8192),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "decode", "decode", "decode", "prefill"])
    rank = rng.choice([128, 256, 384, 512, 512, 512])
    page = rng.choice([1, 16, 16, 24, 32, 48, 64, 64, 128])
    if op in ("append", "read"):
        hi = _log(rng, 1, 4096)
        lo = hi if hi == 1 else rng.randint(0, hi)
        reqs = max(1, min(512, _log(rng, 1, 512), 50000 // max(1, (lo + hi) // 2)))
        if op == "read":
            return dict(op=op, rank=rank, page=page, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), reqs=reqs,
                        len_lo=lo, len_hi=hi)
        return dict(op=op, rank=rank, page=page, rope=rng.random() < 0.9, interleaved=rng.random() < 0.4,
                    norm=rng.random() < 0.8, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), own_pos=rng.random() < 0.6,
                    reqs=reqs, new_lo=lo, new_hi=hi, ctx_lo=0, ctx_hi=min(_log(rng, 1, 4000), 600000 // reqs))
    if op == "prefill":
        heads = rng.choice([1, 3, 8, 16, 32])
        reqs = _log(rng, 1, 24)
        # the products of all heads stay under those of the largest listed case
        length = min(8192, int(math.sqrt(1.0e9 / heads / reqs)))
        hi = _log(rng, 1, length)
        cached = rng.choice([0, 0, 1]) * _log(rng, 1, max(1, length // 2))
        return dict(op=op, heads=heads, causal=rng.random() < 0.8, dtype=rng.choice(["bf16", "bf16", "f16"]), reqs=reqs,
                    len_lo=rng.randint(0, hi), len_hi=hi, cached_hi=cached)
    heads = rng.choice([1, 4, 8, 16, 16, 20, 32, 64, 128])
    nodes = rng.choice([1, 1, 1, 2, 5, 24, 64])
    tree = nodes > 1 and rng.random() < 0.7
    # tokens of all rows, and their products, stay under those of the largest listed cases
    entries = _log(rng, 64, min(900000, 30000000 // (heads * nodes)))
    rows = _log(rng, 1, min(256, entries))
    length = max(nodes, min(entries // rows, 100000))
    topk = nodes == 1 and rng.random() < 0.4
    if topk:
        length = min(length, 2048)
    ctx = length if not topk else max(length, min(_log(rng, length, 20 * length), 32768, max(length, 1000000 // rows)))
    return dict(op=op, rank=rank, page=page, heads=heads, nodes=nodes, topk=length if topk else 0, tree=tree, rows=rows,
                ctx=ctx, len_lo=rng.randint(nodes if nodes > 1 else 0, length), len_hi=length)


# ------------------------------------------------------------------ inputs ----
def _spread(lo, hi, n, gen):
    """n whole numbers from lo to hi, evenly spread, in an order of the seed."""
    x = lo + (torch.arange(n, device="cuda", dtype=torch.float64) * ((hi - lo) / max(1, n - 1))).round()
    return x[torch.randperm(n, generator=gen, device="cuda")].to(torch.int32)


def _spread_list(lo, hi, n):
    return [lo + round(i * ((hi - lo) / max(1, n - 1))) for i in range(n)]


def _cu(counts):
    return torch.cat([torch.zeros_like(counts[:1]), counts.cumsum(0, dtype=torch.int32)])


def _table(length):
    """cos, then sin, of every position's rotation angles, from 64 bits."""
    freq = 500000.0 ** (-torch.arange(0, ROPE, 2, device="cuda", dtype=torch.float64) / ROPE)
    ang = torch.arange(length, device="cuda", dtype=torch.float64)[:, None] * freq
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def _latents(shape, gen):
    """Normal values with a few large channels, as trained projections have them."""
    x = torch.randn(shape, generator=gen, device="cuda")
    return x * (1.0 + 7.0 * (torch.rand(shape[-1], generator=gen, device="cuda") > 0.98))


def _exponent(top):
    """The least e with top <= 448 * 2^e, between the bounds."""
    mant, exp = torch.frexp(top)  # top = mant * 2^exp, mant in [0.5, 1); 448 = 0.875 * 2^9
    e = exp - 9 + (mant > 0.875).to(exp.dtype)
    return torch.where(top > 0, e, E_LOW).clamp(E_LOW, E_HIGH)


def _to_e4m3(x):
    return x.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _filled_cache(pool, page, rank, gen):
    """Caches of tokens with normed latents, some of them small or large."""
    tokens = pool * page
    codes = torch.empty((tokens, rank), dtype=torch.uint8, device="cuda")
    rope = torch.empty((tokens, ROPE), dtype=torch.bfloat16, device="cuda")
    scales = torch.empty(tokens, device="cuda")
    gain = 1.0 + 3.0 * (torch.rand(rank, generator=gen, device="cuda") > 0.98)
    for i in range(0, tokens, 1 << 17):
        n = min(1 << 17, tokens - i)
        x = torch.randn((n, rank), generator=gen, device="cuda") * gain
        x *= torch.exp2(torch.randn((n, 1), generator=gen, device="cuda"))
        s = torch.exp2(_exponent(x.abs().amax(1)).float())
        codes[i:i + n] = _to_e4m3(x / s[:, None]).view(torch.uint8)
        rope[i:i + n] = (torch.randn((n, ROPE), generator=gen, device="cuda") / s[:, None]).to(torch.bfloat16)
        scales[i:i + n] = s
    return (codes.view(torch.float8_e4m3fn).view(pool, page, rank), rope.view(pool, page, ROPE),
            scales.view(pool, page))


def _pages(reqs, per_req, gen):
    """A block table over a shuffled pool with a few spare pages."""
    pool = reqs * per_req + 3
    return torch.randperm(pool, generator=gen, device="cuda")[:reqs * per_req].to(torch.int32).view(reqs, per_req), pool


def _trees(rows, nodes, gen):
    """Ancestor masks, int32 words [rows, nodes, words], of random trees, each node's own bit among them."""
    words = -(-nodes // 32)
    bits = torch.zeros((rows, nodes, words * 32), dtype=torch.bool, device="cuda")
    at = torch.arange(rows, device="cuda")
    for i in range(nodes):
        if i:
            # half of the nodes follow the one before, the others any earlier one
            any_one = torch.randint(0, i, (rows,), generator=gen, device="cuda")
            parent = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.5, any_one, i - 1)
            bits[:, i] = bits[at, parent]
        bits[:, i, i] = True
    value = (bits.view(rows, nodes, words, 32).long() << torch.arange(32, device="cuda")).sum(-1)
    return torch.where(value >= 1 << 31, value - (1 << 32), value).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = dict(case=case)
    if op == "append":
        n, dt = case["reqs"], DTYPES[case["dtype"]]
        count = _spread(case["new_lo"], case["new_hi"], n, gen)
        starts = _spread(case["ctx_lo"], case["ctx_hi"], n, gen)
        total = sum(_spread_list(case["new_lo"], case["new_hi"], n))
        limit = case["ctx_hi"] + case["new_hi"] + 1
        btable, pool = _pages(n, -(-limit // case["page"]), gen)
        packed = _latents((total, case["rank"] + ROPE), gen).to(dt)
        codes, rope, scales = _filled_cache(pool, case["page"], case["rank"], gen)
        s.update(c_new=packed[:, :case["rank"]], r_new=packed[:, case["rank"]:], codes=codes, rope=rope, scales=scales,
                 btable=btable, starts=starts, cu_tokens=None, table=None, positions=None, c_weight=None)
        if not case["new_lo"] == case["new_hi"] == 1:
            s["cu_tokens"] = _cu(count)
        if case["rope"]:
            s["table"] = _table(limit)
            if not case["own_pos"]:
                s["positions"] = torch.randint(0, limit, (total,), generator=gen, device="cuda", dtype=torch.int32)
        if case["norm"]:
            s["c_weight"] = (1 + 0.2 * torch.randn(case["rank"], generator=gen, device="cuda")).to(dt)
    elif op == "read":
        n = case["reqs"]
        count = _spread(case["len_lo"], case["len_hi"], n, gen)
        btable, pool = _pages(n, max(1, -(-case["len_hi"] // case["page"])), gen)
        codes, rope, scales = _filled_cache(pool, case["page"], case["rank"], gen)
        s.update(codes=codes, rope=rope, scales=scales, btable=btable, cu_tokens=_cu(count),
                 starts=torch.zeros(n, dtype=torch.int32, device="cuda"),
                 tokens=sum(_spread_list(case["len_lo"], case["len_hi"], n)))
    elif op == "decode":
        rows, nodes, ctx = case["rows"], case["nodes"], case["ctx"]
        btable, pool = _pages(rows, max(1, -(-ctx // case["page"])), gen)
        codes, rope, scales = _filled_cache(pool, case["page"], case["rank"], gen)
        q = torch.randn((rows, nodes, case["heads"], case["rank"] + ROPE), generator=gen, device="cuda")
        q = q.to(torch.bfloat16)
        s.update(q=q if nodes > 1 else q[:, 0], codes=codes, rope=rope, scales=scales, btable=btable, indices=None,
                 counts=_spread(case["len_lo"], case["len_hi"], rows, gen), tree=None)
        if case["tree"]:
            s["tree"] = _trees(rows, nodes, gen)
        if case["topk"]:
            picks = torch.rand((rows, ctx), generator=gen, device="cuda").argsort(1)[:, :case["topk"]].to(torch.int32)
            past = torch.arange(case["topk"], device="cuda")[None, :] >= s["counts"][:, None]
            s["indices"] = picks.masked_fill_(past, -1).contiguous()
            s["counts"] = None
    else:
        n, heads, dt = case["reqs"], case["heads"], DTYPES[case["dtype"]]
        count = _spread(case["len_lo"], case["len_hi"], n, gen)
        cached = _spread(0, case["cached_hi"], n, gen)
        total = sum(_spread_list(case["len_lo"], case["len_hi"], n))
        keys = total + sum(_spread_list(0, case["cached_hi"], n))
        # the up-projection gives keys and values of a head side by side
        kv = torch.randn((keys, heads, 2 * HEAD), generator=gen, device="cuda").to(dt)
        s.update(q=(1.5 * torch.randn((total, heads, HEAD + ROPE), generator=gen, device="cuda")).to(dt),
                 k=kv[..., :HEAD], v=kv[..., HEAD:],
                 k_rope=torch.randn((keys, ROPE), generator=gen, device="cuda").to(dt),
                 cu_q=_cu(count), cu_k=_cu(count + cached))
        # the bounds on the host, for a loop over the sequences
        s["bounds"] = s["cu_q"].tolist(), s["cu_k"].tolist()
    return s


# ------------------------------------------------------------- plain forms ----
def _slots(s, req, pos):
    page = s["codes"].shape[1]
    return s["btable"].long()[req, pos // page] * page + pos % page


def _token_places(s):
    """Request, place and slot of every token that cu_tokens and starts name."""
    starts = s["starts"].long()
    n = starts.shape[0]
    tokens = s["c_new"].shape[0] if "c_new" in s else s["tokens"]
    cu = s["cu_tokens"].long() if s["cu_tokens"] is not None else torch.arange(n + 1, device=starts.device)
    token = torch.arange(tokens, device=starts.device)
    req = torch.searchsorted(cu, token, right=True) - 1
    pos = starts[req] + token - cu[req]
    return pos, _slots(s, req, pos)


def _rotate(r, table, positions, interleaved):
    r = r.float()
    if table is None:
        return r
    half = ROPE // 2
    cs = table[positions.long()]
    cos, sin = cs[:, :half], cs[:, half:]
    if interleaved:
        a, b = r[:, 0::2], r[:, 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    a, b = r[:, :half], r[:, half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_append(s):
    pos, slot = _token_places(s)
    x = s["c_new"].float()
    if s["c_weight"] is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["c_weight"].float()
    r = _rotate(s["r_new"], s["table"], pos if s["positions"] is None else s["positions"], s["case"]["interleaved"])
    scale = torch.exp2(_exponent(x.abs().amax(-1)).float())
    rank = x.shape[1]
    s["codes"].view(torch.uint8).view(-1, rank)[slot] = _to_e4m3(x / scale[:, None]).view(torch.uint8)
    s["rope"].view(-1, ROPE)[slot] = (r / scale[:, None]).to(torch.bfloat16)
    s["scales"].view(-1)[slot] = scale
    return s["codes"], s["rope"], s["scales"]


def _gathered(s, slot):
    """Latent and rotated part of the tokens at these slots, in 32 bits."""
    rank = s["codes"].shape[2]
    scale = s["scales"].view(-1)[slot][..., None]
    codes = s["codes"].view(torch.uint8).view(-1, rank)[slot].view(torch.float8_e4m3fn).float()
    return codes * scale, s["rope"].view(-1, ROPE)[slot].float() * scale


def _plain_read(s):
    c, r = _gathered(s, _token_places(s)[1])
    dt = DTYPES[s["case"]["dtype"]]
    return c.to(dt), r.to(dt)


def _seen(s, t):
    """Which of the tokens t[rows, T] each row's nodes see: [rows, nodes, T]."""
    nodes = s["case"]["nodes"]
    node = torch.arange(nodes, device=t.device)[None, :, None]
    own_from = s["counts"].long()[:, None, None] - nodes
    d = t[:, None, :] - own_from
    if s["tree"] is None:
        return (d <= node) & (d < nodes)
    word = s["tree"].long()
    at = d.clamp(0, nodes - 1).expand(-1, nodes, -1)
    bit = (torch.gather(word, 2, at // 32) >> (at % 32)) & 1
    return (d < 0) | ((d < nodes) & (bit == 1))


def _plain_decode(s):
    case = s["case"]
    rows, nodes, heads, rank = case["rows"], case["nodes"], case["heads"], case["rank"]
    q = s["q"].float().view(rows, nodes * heads, rank + ROPE)
    if s["indices"] is None:
        t = torch.arange(case["ctx"], device=q.device)[None, :].expand(rows, -1)
        ok = _seen(s, t)
        t = torch.where(ok.any(1), t, 0)
    else:
        t = s["indices"].long()
        ok = (t >= 0)[:, None]
        t = torch.where(t >= 0, t, 0)
    slot = _slots(s, torch.arange(rows, device=q.device)[:, None], t)
    c, r = _gathered(s, slot)
    score = (torch.matmul(q[..., :rank], c.transpose(1, 2)) + torch.matmul(q[..., rank:], r.transpose(1, 2))) * SCALE
    del r
    score = score.view(rows, nodes, heads, -1)
    score = torch.where(ok[:, :, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    del score
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = torch.matmul(p.view(rows, nodes * heads, -1), c).to(torch.bfloat16)
    return out.view(*s["q"].shape[:-1], rank)


def _plain_prefill(s):
    q, k, v, k_rope = s["q"], s["k"], s["v"], s["k_rope"]
    tokens, heads = q.shape[:2]
    out = torch.empty((tokens, heads, HEAD), dtype=q.dtype, device=q.device)
    reqs = s["case"]["reqs"]
    cu_q, cu_k = s["bounds"]
    for e in range(reqs):
        a, b, c, d = cu_q[e], cu_q[e + 1], cu_k[e], cu_k[e + 1]
        if a == b:
            continue
        rope = k_rope[c:d].float().t()
        later = torch.arange(d - c, device=q.device)[None, :] > torch.arange(b - a, device=q.device)[:, None] + (d - c - b + a)
        for h in range(heads):
            x = q[a:b, h].float()
            score = (x[:, :HEAD] @ k[c:d, h].float().t() + x[:, HEAD:] @ rope) * SCALE
            if s["case"]["causal"]:
                score = torch.where(later, -math.inf, score)
            p = torch.exp(score - score.amax(-1, keepdim=True))
            out[a:b, h] = ((p @ v[c:d, h].float()) / p.sum(-1, keepdim=True)).to(q.dtype)
    return out


def run(state):
    s = state
    case = s["case"]
    op = case["op"]
    if not own:
        return {"append": _plain_append, "read": _plain_read, "decode": _plain_decode, "prefill": _plain_prefill}[op](s)
    qsa = _package()
    if op == "append":
        return qsa.qsa_latent_append(s["c_new"], s["r_new"], s["codes"], s["rope"], s["scales"], s["btable"], s["starts"],
                                     cu_tokens=s["cu_tokens"], table=s["table"], positions=s["positions"],
                                     c_weight=s["c_weight"], eps=EPS, interleaved=case["interleaved"])
    if op == "read":
        return qsa.qsa_latent_read(s["codes"], s["rope"], s["scales"], s["btable"], s["starts"], s["cu_tokens"],
                                   s["tokens"], dtype=DTYPES[case["dtype"]])
    if op == "decode":
        return qsa.qsa_latent_decode(s["q"], s["codes"], s["rope"], s["scales"], s["btable"], None, s["indices"],
                                     counts=s["counts"], tree=s["tree"], softmax_scale=SCALE)
    return qsa.qsa_latent_prefill(s["q"], s["k"], s["k_rope"], s["v"], s["cu_q"], s["cu_k"], causal=case["causal"],
                                  softmax_scale=SCALE)


# ------------------------------------------------------------------- work ----
def work(case):
    op = case["op"]
    size = {"bf16": 2, "f16": 2, "f32": 4}.get(case.get("dtype"), 2)
    if op == "prefill":
        lens = _spread_list(case["len_lo"], case["len_hi"], case["reqs"])
        cached = _spread_list(0, case["cached_hi"], case["reqs"])
        tokens, keys, heads = sum(lens), sum(lens) + sum(cached), case["heads"]
        mean_cached = sum(cached) / case["reqs"]
        pairs = sum(n * (n + 1) / 2 + n * mean_cached if case["causal"] else n * (n + mean_cached) for n in lens)
        return {"bytes": size * (tokens * heads * (2 * HEAD + ROPE) + keys * (heads * 2 * HEAD + ROPE)),
                "flops": 2.0 * pairs * heads * (2 * HEAD + ROPE)}
    rank = case["rank"]
    token = rank + 2 * ROPE + 4
    if op == "append":
        tokens = sum(_spread_list(case["new_lo"], case["new_hi"], case["reqs"]))
        return {"bytes": tokens * (size * (rank + ROPE) + token + (4 * ROPE if case["rope"] else 0)) + 8 * case["reqs"],
                "flops": 8.0 * tokens * (rank + ROPE)}
    if op == "read":
        tokens = sum(_spread_list(case["len_lo"], case["len_hi"], case["reqs"]))
        return {"bytes": tokens * (token + size * (rank + ROPE)) + 8 * case["reqs"], "flops": 1.0 * tokens * (rank + ROPE)}
    entries = sum(_spread_list(case["len_lo"], case["len_hi"], case["rows"]))
    queries = case["rows"] * case["nodes"] * case["heads"]
    return {"bytes": entries * (token + (4 if case["topk"] else 0)) + queries * 2 * (2 * rank + ROPE),
            "flops": 2.0 * entries * case["nodes"] * case["heads"] * (2 * rank + ROPE)}


# ------------------------------------------------------------ in 64 bits ----
def _round_e4m3(x):
    """The nearest E4M3FN value, ties to even, saturated, in 64 bits."""
    a = x.abs().clamp_max(E4M3_MAX)
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3)
    return torch.round(a / step) * step * x.sign()


def _request_slots(s, e, first, count):
    page = s["codes"].shape[1]
    pos = torch.arange(first, first + count, device="cuda")
    return pos, s["btable"][e].long()[torch.div(pos, page, rounding_mode="floor")] * page + torch.remainder(pos, page)


def _bounds(s):
    n = s["starts"].shape[0]
    return s["cu_tokens"].tolist() if s["cu_tokens"] is not None else list(range(n + 1))


def _exact_append(s):
    case = s["case"]
    rank = case["rank"]
    cu, starts = _bounds(s), s["starts"].tolist()
    places = [_request_slots(s, e, starts[e], cu[e + 1] - cu[e]) for e in range(len(starts))]
    pos, slot = torch.cat([p for p, _ in places]), torch.cat([x for _, x in places])
    x = s["c_new"].double()
    if s["c_weight"] is not None:
        x = x / ((x ** 2).sum(-1, keepdim=True) / rank + EPS).sqrt() * s["c_weight"].double()
    r = s["r_new"].double()
    if s["table"] is not None:
        at = pos if s["positions"] is None else s["positions"].long()
        half = ROPE // 2
        turn = torch.complex(s["table"][at, :half].double(), s["table"][at, half:].double())
        first, second = (r[:, 0::2], r[:, 1::2]) if case["interleaved"] else (r[:, :half], r[:, half:])
        z = torch.complex(first, second) * turn
        r = torch.view_as_real(z).flatten(1) if case["interleaved"] else torch.cat([z.real, z.imag], 1)
    top = x.abs().amax(1)
    e = torch.ceil(torch.log2((top / E4M3_MAX).clamp_min(2.0 ** -200))).clamp(E_LOW, E_HIGH)
    scale = torch.exp2(e)[:, None]
    codes, rope = s["codes"].double().view(-1, rank), s["rope"].double().view(-1, ROPE)
    scales = s["scales"].double().view(-1)
    codes[slot] = _round_e4m3(x / scale)
    rope[slot] = r / scale
    scales[slot] = scale[:, 0]
    return codes.view(s["codes"].shape), rope.view(s["rope"].shape), scales.view(s["scales"].shape)


def _exact_values(s, slot):
    rank = s["codes"].shape[2]
    scale = s["scales"].view(-1)[slot].double()[:, None]
    codes = s["codes"].view(torch.uint8).view(-1, rank)[slot].view(torch.float8_e4m3fn).double()
    return codes * scale, s["rope"].view(-1, ROPE)[slot].double() * scale


def _exact_read(s):
    cu, starts = _bounds(s), s["starts"].tolist()
    slot = torch.cat([_request_slots(s, e, starts[e], cu[e + 1] - cu[e])[1] for e in range(len(starts))])
    return _exact_values(s, slot)


def _exact_decode(s):
    case = s["case"]
    rows, nodes, heads, rank, page = (case[x] for x in ("rows", "nodes", "heads", "rank", "page"))
    q = s["q"].view(rows, nodes, heads, rank + ROPE)
    out = torch.zeros((rows, nodes, heads, rank), dtype=torch.float64, device=q.device)
    counts = s["counts"].tolist() if s["indices"] is None else (s["indices"] >= 0).sum(1).tolist()
    tree = s["tree"].cpu().numpy() if s["tree"] is not None else None
    for e in range(rows):
        if not counts[e]:
            continue
        if s["indices"] is None:
            slot = _request_slots(s, e, 0, counts[e])[1]
        else:
            t = s["indices"][e, :counts[e]].long()
            slot = s["btable"][e].long()[t // page] * page + t % page
        c, r = _exact_values(s, slot)
        score = torch.einsum("nhd,td->nht", q[e].double(), torch.cat([c, r], 1)) * SCALE
        if nodes > 1:
            hidden = torch.zeros((nodes, nodes), dtype=torch.bool)
            for i in range(nodes):
                for j in range(nodes):
                    hidden[i, j] = j > i if tree is None else not (int(tree[e, i, j // 32]) >> (j % 32)) & 1
            score[:, :, counts[e] - nodes:].masked_fill_(hidden.to(q.device)[:, None], -math.inf)
        out[e] = torch.einsum("nht,td->nhd", torch.softmax(score, -1), c)
    return out.view(*s["q"].shape[:-1], rank)


def _exact_prefill(s):
    q, heads = s["q"], s["case"]["heads"]
    out = torch.zeros((*q.shape[:2], HEAD), dtype=torch.float64, device=q.device)
    cu_q, cu_k = s["cu_q"].tolist(), s["cu_k"].tolist()
    for e in range(len(cu_q) - 1):
        n, m = cu_q[e + 1] - cu_q[e], cu_k[e + 1] - cu_k[e]
        k_rope = s["k_rope"][cu_k[e]:cu_k[e + 1]].double()
        for h in range(heads if n else 0):
            key = torch.cat([s["k"][cu_k[e]:cu_k[e + 1], h].double(), k_rope], 1)
            for i in range(0, n, 2048):
                score = q[cu_q[e] + i:min(cu_q[e] + i + 2048, cu_q[e + 1]), h].double() @ key.t() / math.sqrt(HEAD + ROPE)
                if s["case"]["causal"]:
                    score = score.masked_fill(torch.ones_like(score, dtype=torch.bool).triu(m - n + i + 1), -math.inf)
                out[cu_q[e] + i:cu_q[e] + i + len(score), h] = (
                    torch.softmax(score, -1) @ s["v"][cu_k[e]:cu_k[e + 1], h].double())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "read": _exact_read, "decode": _exact_decode, "prefill": _exact_prefill}[case["op"]](s)
