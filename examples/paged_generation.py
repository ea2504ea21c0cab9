"""A small generation loop over the paged cache, its attention and the MoE layers, as a serving program runs them.

    python examples/paged_generation.py [--prompts 2] [--samples 2] [--steps 8]

A model of random weights (attention + routed-expert MoE per layer) reads ragged prompts (``extend``, ``write``,
``attn_prefill``), forks each into samples that share the prompt's full pages (``fork``), decodes them together
(``extend``, ``write``, ``attn_decode``, ``moe_layer_decode``), drops half of them and packs the pool (``free``,
``compact``) and goes on. Nothing in a step waits for the host but the final read of the tokens.
"""
import argparse
import sys
from pathlib import Path

import numpy as np
import torch

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT / "slotstream-spark_b200"))

from slotstream_b200 import synth  # noqa: E402
from slotstream_b200.kernels.moe_layer import DecodeLayerBuffers, moe_layer_decode  # noqa: E402
from slotstream_b200.kernels.paged_attention import attn_decode, attn_prefill  # noqa: E402
from slotstream_b200.kv_cache import PagedKvCache  # noqa: E402
from slotstream_b200.records import EXPERTS_PER_LAYER, MAP_LAYERS, RecordLayout  # noqa: E402


class Model:
    """Random weights: per layer a fused q/k/v projection, an output projection and a routed-expert MoE layer."""

    def __init__(self, layers=2, hidden=512, inter=512, experts=16, topk=4, heads=8, kv_heads=2, head_dim=64, vocab=1024,
                 window=0, sinks=0, seed=0):
        self.layers, self.hidden, self.heads, self.kv, self.dim = layers, hidden, heads, kv_heads, head_dim
        self.topk, self.experts, self.inter, self.window, self.sinks = topk, experts, inter, window, sinks
        lay = RecordLayout(hidden, inter)
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(*shape):
            return (torch.randn(*shape, device="cuda", generator=g) * shape[-1] ** -0.5).to(torch.bfloat16)

        def bits(a):
            return torch.from_numpy(np.ascontiguousarray(a).view(np.int16)).view(torch.bfloat16).cuda()

        self.embed, self.head = weight(vocab, hidden) * hidden ** 0.5, weight(vocab, hidden)
        self.qkv = [weight((heads + 2 * kv_heads) * head_dim, hidden) for _ in range(layers)]
        self.proj = [weight(hidden, heads * head_dim) for _ in range(layers)]
        self.router = [bits(synth.router_weight(seed, experts, hidden, l)) for l in range(layers)]
        self.gate = [bits(synth.shared_gate_weight(seed, hidden, l)) for l in range(layers)]
        recs = [np.stack([synth.expert_record(lay, seed, l, e) for e in range(experts + 1)]) for l in range(layers)]
        self.records = torch.from_numpy(np.stack(recs)).cuda()
        size = lay.record_bytes
        self.slots = torch.tensor([self.records.data_ptr() + i * size for i in range(layers * (experts + 1))], device="cuda")
        m = torch.full((MAP_LAYERS * EXPERTS_PER_LAYER,), -1, dtype=torch.int32)
        for l in range(layers):
            m[l * EXPERTS_PER_LAYER:l * EXPERTS_PER_LAYER + experts] = torch.arange(experts, dtype=torch.int32) + l * (experts + 1)
        self.map = m.cuda()

    def _norm(self, x):
        return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6)).to(torch.bfloat16)

    def forward(self, cache, tokens, starts, ids, decode: bool):
        """Logits of every row of ``tokens``, whose keys and values go into the cache (which ``extend`` made room for)."""
        x, rows = self.embed[tokens], tokens.numel()
        for l in range(self.layers):
            qkv = (self._norm(x) @ self.qkv[l].t()).view(rows, -1, self.dim)
            q, k, v = qkv.split([self.heads, self.kv, self.kv], 1)
            cache.write(l, k, v, starts, ids)
            kw = dict(ids=ids, window=self.window, sinks=self.sinks, err=cache.err)
            if decode:
                o = attn_decode(q[:, None], cache.k(l), cache.v(l), cache.table, cache.lengths, **kw)
            else:
                o = attn_prefill(q, cache.k(l), cache.v(l), cache.table, cache.lengths, starts, **kw)
            x = x + o.reshape(rows, -1) @ self.proj[l].t()
            bufs = DecodeLayerBuffers(rows, self.topk, self.hidden, self.inter, self.experts)
            x = x + moe_layer_decode(self._norm(x), self.router[l], l, self.map, self.slots, self.records[l, self.experts],
                                     self.gate[l], self.topk, bufs)
        return (self._norm(x) @ self.head.t()).float()


def generate(model, prompts, samples: int, steps: int, page_size: int = 16, clone=None):
    """Greedy continuations: sample s of a prompt starts with its s-th best token. After half the steps every other
    sequence is dropped and the pool is packed. Returns (tokens [sequences kept, steps], logits of the last step, cache).
    ``clone(cache, parents, children)`` replaces the fork (tests)."""
    n, longest = len(prompts), max(len(p) for p in prompts) + steps
    seqs, max_pages = n * samples, -(-longest // page_size)
    cache = PagedKvCache(seqs * (max_pages + 1), model.layers, model.kv, page_size, model.dim, seqs, max_pages)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    firsts = list(range(0, seqs, samples))
    lens = [len(p) for p in prompts]
    starts, ids = ints([0] + np.cumsum(lens).tolist()), ints(firsts)
    cache.extend(ids, ints(lens))
    logits = model.forward(cache, torch.cat([torch.as_tensor(p, device="cuda") for p in prompts]), starts, ids, decode=False)
    best = logits[starts[1:].long() - 1].topk(samples, -1).indices               # [n, samples]
    if samples > 1:
        parents = ints([f for f in firsts for _ in range(samples - 1)])
        children = ints([f + s for f in firsts for s in range(1, samples)])
        (clone or PagedKvCache.fork)(cache, parents, children)
    live, token, out = ints(range(seqs)), best.reshape(-1), []
    for step in range(steps):
        if step == steps // 2 and seqs > 1:
            cache.free(live[1::2].contiguous())
            cache.compact()
            keep = torch.arange(0, live.numel(), 2, device="cuda")
            live, token, out = live[keep], token[keep], [t[keep] for t in out]
        out.append(token)
        m = live.numel()
        cache.extend(live, torch.ones(m, dtype=torch.int32, device="cuda"))
        logits = model.forward(cache, token, torch.arange(m + 1, dtype=torch.int32, device="cuda"), live, decode=True)
        token = logits.argmax(-1)
    cache.check()
    return torch.stack(out, 1), logits, cache


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--prompts", type=int, default=2)
    ap.add_argument("--samples", type=int, default=2)
    ap.add_argument("--steps", type=int, default=8)
    a = ap.parse_args()
    r = np.random.default_rng(0)
    prompts = [r.integers(0, 1024, int(r.integers(5, 200))).tolist() for _ in range(a.prompts)]
    tokens, _, cache = generate(Model(), prompts, a.samples, a.steps)
    for i, t in enumerate(tokens.tolist()):
        print(f"sequence {i}: {t}")
    used = int((cache.refs > 0).sum())
    print(f"{used} of {cache.pages} pages in use, {int((cache.refs > 1).sum())} shared")


if __name__ == "__main__":
    main()
