"""A small serving loop over the block-scaled cache.

    python examples/block_cache_serving.py [--requests 8] [--steps 4] [--topk 64]

One attention layer: the prompts of a few requests are appended to the paged
cache in one call, then every step takes one token of each request: its
projected queries, keys and values are normed, rotated and appended, and the
queries attend, over the whole context and over the Top-K positions that an
indexer's scores pick. The last step is compared with a plain fp32 computation
of the same attention from the projections.
"""

from __future__ import annotations

import argparse
import sys
from dataclasses import dataclass
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "qsa-fp8-sm89_b200"))

import qsa_b200 as qsa  # noqa: E402

D = 128


@dataclass
class Layer:
    """What a model keeps for one attention layer and its cache."""

    hq: int
    hkv: int
    table: torch.Tensor     # rotation
    q_weight: torch.Tensor  # head norms
    k_weight: torch.Tensor
    btable: torch.Tensor
    cache: tuple            # k_cache, v_cache, k_scales, v_scales

    def split(self, qkv):
        return qkv[:, :self.hq], qkv[:, self.hq:self.hq + self.hkv], qkv[:, self.hq + self.hkv:]

    def append(self, qkv, starts, cu_tokens=None):
        _, k, v = self.split(qkv)
        qsa.qsa_block_append(k, v, *self.cache, self.btable, starts, cu_tokens=cu_tokens, table=self.table,
                             k_weight=self.k_weight)

    def step(self, qkv, lengths, gate, indices=None):
        """One token of every request: ``lengths`` tokens are cached before it."""
        q, _, _ = self.split(qkv)
        q, _ = qsa.qsa_qk_rope(q, None, self.table, lengths, q_weight=self.q_weight)
        self.append(qkv, lengths)
        if indices is None:
            return qsa.qsa_block_decode(q, *self.cache, self.btable, None, gate=gate, counts=lengths + 1)
        return qsa.qsa_block_decode(q, *self.cache, self.btable, None, indices, gate=gate)


def plain(layer, history, positions, qkv, position, gate, picks=None):
    """The same attention of one request in fp32, from its projections."""
    def turned(x, weight, pos):
        x = x.float() * torch.rsqrt(x.float().pow(2).mean(-1, keepdim=True) + 1e-6) * weight.float()
        c, s = layer.table[pos][:, None, :D // 2], layer.table[pos][:, None, D // 2:]
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    q, _, _ = layer.split(qkv)
    _, k, v = layer.split(history)
    q, k, v = turned(q, layer.q_weight, position[None])[0], turned(k, layer.k_weight, positions), v.float()
    if picks is not None:
        k, v = k[picks], v[picks]
    group = layer.hq // layer.hkv
    score = torch.einsum("hd,thd->ht", q, k.repeat_interleave(group, 1)) * D ** -0.5
    out = torch.einsum("ht,thd->hd", score.softmax(-1), v.repeat_interleave(group, 1))
    return out * torch.sigmoid(gate.float())


def serve(requests=8, steps=4, topk=64, hq=32, hkv=8, page=16, block=16, seed=0, device="cuda"):
    """Runs the loop; returns the largest errors of the dense and the sparse
    outputs of the last step against ``plain``, relative to their rms."""
    gen = torch.Generator(device=device).manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=gen, device=device)
    prompt = torch.randint(1, 300, (requests,), generator=gen, device=device, dtype=torch.int32)
    pages_per_req = -(-(300 + steps) // page)
    pages = requests * pages_per_req
    layer = Layer(
        hq, hkv, qsa.rope_table(300 + steps, D, 500000.0, device=device),
        (1 + 0.1 * rand(D)).to(torch.bfloat16), (1 + 0.1 * rand(D)).to(torch.bfloat16),
        torch.randperm(pages, generator=gen, device=device).to(torch.int32).view(requests, pages_per_req),
        qsa.block_cache(pages, page, hkv, block, device=device))

    cu = torch.cat([torch.zeros_like(prompt[:1]), prompt.cumsum(0, dtype=torch.int32)])
    heads = hq + 2 * hkv
    prompts = rand(int(cu[-1]), heads, D).to(torch.bfloat16)
    layer.append(prompts, torch.zeros_like(prompt), cu)
    history = [prompts[int(a):int(b)] for a, b in zip(cu, cu[1:])]

    lengths = prompt.clone()
    for _ in range(steps):
        qkv, gate = rand(requests, heads, D).to(torch.bfloat16), rand(requests, hq, D).to(torch.bfloat16)
        scores = rand(requests, pages_per_req * page)  # an indexer's, one per position
        picks = qsa.qsa_topk_select(scores, topk, lengths=lengths + 1)
        dense = layer.step(qkv, lengths, gate)
        sparse = layer.step(qkv, lengths, gate, picks)  # the same token once more: the cache stays as it is
        history = [torch.cat([h, qkv[r:r + 1]]) for r, h in enumerate(history)]
        lengths = lengths + 1

    errors = []
    for out, chosen in ((dense, None), (sparse, picks)):
        worst = 0.0
        for r, h in enumerate(history):
            at = None if chosen is None else chosen[r][chosen[r] >= 0].long()
            ref = plain(layer, h, torch.arange(len(h), device=device), qkv[r:r + 1], lengths[r].long() - 1, gate[r], at)
            worst = max(worst, float((out[r].float() - ref).norm() / ref.norm()))
        errors.append(worst)
    return errors


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--steps", type=int, default=4)
    ap.add_argument("--topk", type=int, default=64)
    args = ap.parse_args(argv)
    dense, sparse = serve(args.requests, args.steps, args.topk)
    print(f"relative error against fp32 from the projections: {dense:.3f} (whole contexts), {sparse:.3f} (Top-K)")


if __name__ == "__main__":
    main()
