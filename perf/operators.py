"""Workloads of the paged key-value cache and the attention that reads it.

Four operators, as a serving loop around the MoE layers uses them:

* ``decode`` -- attention of each sequence's newest tokens over its cached pages (one token of a decode step, or the
  two to four of a speculative verify), with an optional sliding window and first tokens that stay visible;
* ``prompt`` -- attention of ragged prompt chunks over their pages, causal, with the same window and sinks;
* ``append`` -- pages allocated for new tokens, and the tokens' keys and values written into them;
* ``pages``  -- sequences forked (full pages shared, the last partial one copied), freed and the pool compacted.

``run`` computes a case with elementary torch operations in 32 bits, or, where ``own`` is true, with the calls that a
user makes of this repository's package.

The cache of a case: ``pool`` [pages, layers, 2, kv_heads, page, dim] (keys at 0, values at 1) and one int32 tensor
``meta`` holding, in this order, lengths [seqs], refs [pages] (tables that hold a page), free words [ceil(pages / 32)]
(bit p % 32 of word p / 32 is set while page p is free), table [seqs, max_pages] (-1 where there is no page) and one
error word."""
import math
import sys

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
PACKAGE = "slotstream-spark_b200"


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # One user's token at a short context: the smallest decode call, where the launch counts.
        dict(name="decode_one_2k", op="decode", dtype="bf16", seqs=1, q_len=1, heads=16, kv_heads=2, dim=256, page=16,
             max_len=2048, ragged=False, window=0, sinks=0),
        # One user's token at the 131,072-token context of the streaming workload.
        dict(name="decode_one_131k", op="decode", dtype="bf16", seqs=1, q_len=1, heads=16, kv_heads=2, dim=256,
             page=16, max_len=131072, ragged=False, window=0, sinks=0),
        # A loaded server's step: 64 sequences of very different lengths (one of them still empty).
        dict(name="decode_batch_ragged", op="decode", dtype="fp16", seqs=64, q_len=1, heads=32, kv_heads=8, dim=128,
             page=32, max_len=16384, ragged=True, window=0, sinks=0),
        # Speculative verify of two tokens for 16 sequences through a windowed layer; the page is no power of two.
        dict(name="verify_window", op="decode", dtype="bf16", seqs=16, q_len=2, heads=24, kv_heads=8, dim=64, page=24,
             max_len=30000, ragged=True, window=1024, sinks=4),
        # A few short prompts admitted together: the smallest prompt call.
        dict(name="prompt_short", op="prompt", dtype="fp16", seqs=5, new=129, ragged=True, ctx=0, heads=8, kv_heads=2,
             dim=64, page=16, window=0, sinks=0),
        # Two users' 2,048-token chunks over long cached contexts, full causal attention.
        dict(name="prompt_chunk_ctx", op="prompt", dtype="bf16", seqs=2, new=2048, ragged=False, ctx=30001, heads=16,
             kv_heads=2, dim=256, page=16, window=0, sinks=0),
        # A whole 32,768-token prompt through a sliding-window layer with sinks.
        dict(name="prompt_32k_window", op="prompt", dtype="bf16", seqs=1, new=32768, ragged=False, ctx=0, heads=32,
             kv_heads=8, dim=128, page=64, window=4096, sinks=16),
        # The cache writes of one decode step of 16 tokens, one layer.
        dict(name="append_step", op="append", dtype="bf16", seqs=16, new=1, ragged=False, ctx=1023, kv_heads=2,
             dim=256, page=16),
        # The cache writes of 32,768 prompt tokens in four ragged prompts, one layer.
        dict(name="append_prompts", op="append", dtype="bf16", seqs=4, new=16384, ragged=True, ctx=77, kv_heads=8,
             dim=128, page=32),
        # One beam split off a short sequence of a one-layer cache: the smallest page call.
        dict(name="fork_one", op="pages", kind="fork", dtype="bf16", layers=1, seqs=1, children=1, kv_heads=2, dim=256,
             page=16, max_len=600),
        # Seven samples branched off each of 16 prompts, 48 layers a page.
        dict(name="fork_samples", op="pages", kind="fork", dtype="bf16", layers=48, seqs=16, children=7, kv_heads=2,
             dim=256, page=16, max_len=600),
        # Half of 24 sequences finished: their pages freed and the pool packed, 48 layers a page.
        dict(name="retire_half", op="pages", kind="retire", dtype="bf16", layers=48, seqs=24, children=0, kv_heads=2,
             dim=256, page=16, max_len=900),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _shape(rng):
    kv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 8, 16])
    return dict(dtype=rng.choice(["bf16", "fp16"]), heads=kv * group, kv_heads=kv, dim=rng.choice([64, 128, 256]),
                page=rng.choice([8, 12, 16, 16, 24, 32, 64, 100, 128]))


def _mask(rng):
    if rng.random() < 0.5:
        return dict(window=0, sinks=0)
    return dict(window=_log(rng, 1, 8192), sinks=rng.choice([0, 1, 4, 16, 100]))


def draw(rng):
    op = rng.choice(["decode", "decode", "prompt", "prompt", "append", "pages"])
    top = {o: max(_cost(c) for c in listed() if c["op"] == o) for o in ("decode", "prompt", "append", "pages")}
    while True:
        if op == "decode":
            c = dict(op=op, seqs=_log(rng, 1, 64), q_len=rng.choice([1, 1, 2, 3, 4]), max_len=_log(rng, 1, 131072),
                     ragged=rng.random() < 0.7, **_shape(rng), **_mask(rng))
            fits = c["seqs"] * c["max_len"] * c["kv_heads"] * c["dim"] <= 64 * 16384 * 8 * 128
        elif op == "prompt":
            c = dict(op=op, seqs=_log(rng, 1, 16), new=_log(rng, 1, 32768), ragged=rng.random() < 0.6,
                     ctx=rng.choice([0, 0, _log(rng, 1, 32768)]), **_shape(rng), **_mask(rng))
            fits = c["seqs"] * c["new"] <= 32768 and c["seqs"] * (c["new"] + c["ctx"]) <= 65536
        elif op == "append":
            s = _shape(rng)
            s.pop("heads")
            c = dict(op=op, seqs=_log(rng, 1, 64), new=_log(rng, 1, 16384), ragged=rng.random() < 0.6,
                     ctx=_log(rng, 1, 4096), **s)
            fits = c["seqs"] * (c["new"] + c["ctx"]) <= 65536
        else:
            s = _shape(rng)
            s.pop("heads")
            kind = rng.choice(["fork", "retire"])
            c = dict(op=op, kind=kind, layers=rng.choice([1, 4, 48]), seqs=_log(rng, 1, 24) + (kind == "retire"),
                     children=_log(rng, 1, 7) if kind == "fork" else 0, max_len=_log(rng, 1, 900), **s)
            fits = _pages_of(c)["pages"] * _page_bytes(c) <= 1800 << 20
        if fits and _cost(c) <= top[op]:
            return c


# ------------------------------------------------------------------------------------------------ sizes of a case
def _spread(i):
    return ((i + 1) * 0.6180339887498949) % 1.0


def _lens(case):
    """(cached lengths before the call, new tokens) of every sequence; they follow from the case alone."""
    n = case["seqs"]
    if case["op"] == "decode":
        full = [1 + int((case["max_len"] - 1) * _spread(i) ** 2) if case["ragged"] else case["max_len"]
                for i in range(n)]
        full[0] = case["max_len"]
        if case["ragged"] and n >= 8:
            full[n // 2] = 0
        return [max(0, t - case["q_len"]) for t in full], [min(t, case["q_len"]) for t in full]
    new = [1 + int((case["new"] - 1) * _spread(i)) if case["ragged"] else case["new"] for i in range(n)]
    new[-1] = case["new"]
    return [int(case["ctx"] * _spread(i + 3)) if case["ctx"] > 1 else case["ctx"] for i in range(n)], new


def _pages_of(case):
    """A page case's lengths, its pages (dealt round the sequences in turn, as they grow together) and pool size."""
    ps, n = case["page"], case["seqs"]
    lens = [1 + int((case["max_len"] - 1) * _spread(i)) for i in range(n)]
    held = [-(-t // ps) for t in lens]
    rows, nxt = [[] for _ in range(n)], 0
    for j in range(max(held)):
        for i in range(n):
            if j < held[i]:
                rows[i].append(nxt)
                nxt += 1
    return dict(lens=lens, rows=rows, used=nxt, pages=nxt + n * case["children"] + 5)


def _page_bytes(case):
    return case.get("layers", 1) * 2 * case["kv_heads"] * case["page"] * case["dim"] * 2


def _visible(lens, new, window, sinks):
    """(query, token) pairs that attend, and tokens that some query of the sequence sees, over all sequences."""
    pairs = tokens = 0
    for c, n in zip(lens, new):
        p = np.arange(c, c + n, dtype=np.int64)
        if window:
            pairs += int(np.minimum(p + 1, window + np.minimum(sinks, np.maximum(p + 1 - window, 0))).sum())
            tokens += min(c + n, window + n - 1 + min(sinks, max(c - window + 1, 0))) if n else 0
        else:
            pairs += int((p + 1).sum())
            tokens += c + n if n else 0
    return pairs, tokens


def work(case):
    if case["op"] in ("decode", "prompt"):
        lens, new = _lens(case)
        pairs, tokens = _visible(lens, new, case["window"], case["sinks"])
        rows = (case["seqs"] * case["q_len"] if case["op"] == "decode" else sum(new)) * case["heads"]
        table = sum(-(-(c + n) // case["page"]) for c, n in zip(lens, new)) if not case["window"] else 0
        return {"bytes": tokens * case["kv_heads"] * case["dim"] * 4 + rows * (case["dim"] * 4 + 4) + table * 4,
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    if case["op"] == "append":
        lens, new = _lens(case)
        return {"bytes": sum(new) * case["kv_heads"] * case["dim"] * 8, "flops": 0}
    p = _pages_of(case)
    if case["kind"] == "fork":
        moved = sum(1 for t in p["lens"] if t % case["page"]) * case["children"]
        table = sum(len(r) for r in p["rows"]) * case["children"]
    else:
        kept = sorted(x for i, r in enumerate(p["rows"]) if i % 2 for x in r)
        moved, table = sum(1 for x in kept if x >= len(kept)), p["used"]
    return {"bytes": 2 * moved * _page_bytes(case) + 8 * table, "flops": 0}


def _cost(case):
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] / 1.5e15


# ------------------------------------------------------------------------------------------------ inputs
def _words(free):
    bits = np.zeros(-(-free.size // 32) * 32, dtype=np.int64)
    bits[:free.size] = free
    return (bits.reshape(-1, 32) << np.arange(32)).sum(1).astype(np.uint32).view(np.int32)


def _meta(lens, rows, pages, max_pages):
    refs, table = np.zeros(pages, np.int32), np.full((len(rows), max_pages), -1, np.int32)
    for i, r in enumerate(rows):
        table[i, :len(r)] = r
        refs[r] += 1
    return np.concatenate([np.array(lens, np.int32), refs, _words(refs == 0), table.reshape(-1), np.zeros(1, np.int32)])


def _split(meta, seqs, pages):
    w = -(-pages // 32)
    a, b, c = seqs, seqs + pages, seqs + pages + w
    return dict(lengths=meta[:a], refs=meta[a:b], words=meta[b:c], table=meta[c:-1].view(seqs, -1), err=meta[-1:])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 11)
    host = np.random.default_rng(seed)
    dt, ps = TYPES[case["dtype"]], case["page"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g, dtype=dt)

    if case["op"] == "pages":
        p = _pages_of(case)
        n, kids = case["seqs"], case["seqs"] * case["children"]
        max_pages = max(len(r) for r in p["rows"]) + 2
        meta = _meta(p["lens"] + [0] * kids, p["rows"] + [[]] * kids, p["pages"], max_pages)
        state = dict(case=case, meta0=torch.from_numpy(meta).cuda(), seqs=n + kids, pages=p["pages"],
                     pool=normal(p["pages"], case["layers"], 2, case["kv_heads"], ps, case["dim"]))
        state["meta"] = state["meta0"].clone()
        which = host.permutation(kids)
        if case["kind"] == "fork":
            state["parents"] = torch.from_numpy((which % n).astype(np.int32)).cuda()
            state["children"] = torch.from_numpy((n + np.arange(kids)).astype(np.int32)).cuda()
        else:
            state["done"] = torch.from_numpy(host.permutation(np.arange(0, n, 2)).astype(np.int32)).cuda()
        return state

    lens, new = _lens(case)
    n = case["seqs"]
    before = lens if case["op"] == "append" else [a + b for a, b in zip(lens, new)]
    held = [-(-t // ps) for t in before]
    total = sum(-(-(a + b) // ps) for a, b in zip(lens, new))
    pages = total + 3
    order = host.permutation(pages)[:sum(held)]
    ends = np.cumsum([0] + held)
    rows = [order[ends[i]:ends[i + 1]] for i in range(n)]
    max_pages = max(max(-(-(a + b) // ps) for a, b in zip(lens, new)), 1) + 1
    meta = torch.from_numpy(_meta(before, rows, pages, max_pages)).cuda()
    pool = normal(pages, 1, 2, case["kv_heads"], ps, case["dim"])
    if case["op"] != "append":
        # what no token was written to holds what was left there, not-a-numbers among it
        tail = torch.from_numpy(np.array([t % ps or ps for t, h in zip(before, held) if h], np.int64)).cuda()
        last = torch.from_numpy(np.array([r[-1] for r in rows if len(r)], np.int64)).cuda()
        dead = torch.arange(ps, device="cuda")[None] >= tail[:, None]
        ends_of = pool[last]
        pool[last] = ends_of.masked_fill(dead[:, None, None, None, :, None], float("nan"))
    starts = torch.from_numpy(np.cumsum([0] + new).astype(np.int32)).cuda()
    state = dict(case=case, pool=pool, seqs=n, pages=pages, lens=lens, new=new, starts=starts)
    if case["op"] == "decode":
        # the projections' output of the step, queries, keys and values side by side; queries of a trained layer are
        # larger than one, so that some tokens stand out
        both = normal(n, case["q_len"], case["heads"] + 2 * case["kv_heads"], case["dim"])
        state.update(meta=meta, q=both[:, :, :case["heads"]].mul_(2))
    elif case["op"] == "prompt":
        both = normal(sum(new), case["heads"] + 2 * case["kv_heads"], case["dim"])
        state.update(meta=meta, q=both[:, :case["heads"]].mul_(2))
    else:
        both = normal(sum(new), 3 * case["kv_heads"], case["dim"])
        kv = case["kv_heads"]
        state.update(meta0=meta, meta=meta.clone(), k=both[:, kv:2 * kv], v=both[:, 2 * kv:],
                     ids=torch.arange(n, dtype=torch.int32, device="cuda"),
                     counts=torch.tensor(new, dtype=torch.int32, device="cuda"))
    return state


# ------------------------------------------------------------------------------------------------ the plain forms
def _attend(q, k, v, at, length, window, sinks):
    """q [.., R, D] at positions `at` [.., R] over k, v [.., L, D] of sequences `length` long -> (o, lse), 32 bits."""
    t = torch.arange(k.shape[-2], device=q.device)
    seen = (t <= at[..., None]) & (t < length)
    if window:
        seen &= (at[..., None] - t < window) | (t < sinks)
    v = torch.where(seen.any(-2)[..., None], v, 0.0)
    s = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(q.shape[-1]))
    s = torch.where(seen, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    o = torch.where(total > 0, (p @ v) / total, 0.0)
    return o, (m + torch.log(total)).squeeze(-1)


def _plain_decode(state):
    case, q = state["case"], state["q"]
    cache = _split(state["meta"], state["seqs"], state["pages"])
    n, ql, heads, d = q.shape
    kv, ps = case["kv_heads"], case["page"]
    t = torch.arange(max(case["max_len"], 1), device=q.device)
    page = cache["table"].long()[:, t // ps].clamp_min(0)                       # [n, L]
    k = state["pool"][page, 0, 0, :, t % ps].float().transpose(1, 2)            # [n, kv, L, d]
    v = state["pool"][page, 0, 1, :, t % ps].float().transpose(1, 2)
    rows = q.float().view(n, ql, kv, heads // kv, d).transpose(1, 2).reshape(n, kv, -1, d)
    length = cache["lengths"].long().view(n, 1, 1)
    at = (length - ql + torch.arange(ql, device=q.device).repeat_interleave(heads // kv)).expand(n, 1, -1)
    o, lse = _attend(rows, k, v, at, length[..., None], case["window"], case["sinks"])
    o = o.view(n, kv, ql, -1, d).transpose(1, 2).reshape(n, ql, heads, d)
    return [o.to(q.dtype), lse.view(n, kv, ql, -1).transpose(1, 2).reshape(n, ql, heads)]


def _plain_prompt(state):
    """Blocks of queries bound the scores' memory (32,768 x 32,768 x heads would not fit)."""
    case, q, ps = state["case"], state["q"], state["case"]["page"]
    kv, (tokens, heads, d) = case["kv_heads"], q.shape
    table = _split(state["meta"], state["seqs"], state["pages"])["table"].long()
    out, lse = torch.empty(tokens, heads, d, dtype=q.dtype, device=q.device), torch.empty(tokens, heads, device=q.device)
    row = 0
    for i, (c, n) in enumerate(zip(state["lens"], state["new"])):
        for a in range(0, n, 1024):
            b = min(a + 1024, n)
            first = max(0, c + a - case["window"] + 1) if case["window"] else 0
            t = torch.arange(first, c + b, device=q.device)
            if first and case["sinks"]:
                t = torch.cat([torch.arange(min(case["sinks"], first), device=q.device), t])
            k = state["pool"][table[i, t // ps], 0, 0, :, t % ps].float().transpose(0, 1)[:, None]   # [kv, 1, L, d]
            v = state["pool"][table[i, t // ps], 0, 1, :, t % ps].float().transpose(0, 1)[:, None]
            x = q[row + a:row + b].float().view(b - a, kv, -1, d).permute(1, 2, 0, 3)                # [kv, G, R, d]
            at = torch.arange(c + a, c + b, device=q.device)[:, None]
            seen = t <= at
            if case["window"]:
                seen &= (at - t < case["window"]) | (t < case["sinks"])
            s = torch.where(seen, (x @ k.transpose(-1, -2)) * (1.0 / math.sqrt(d)), -math.inf)
            m = s.amax(-1, keepdim=True)
            p = torch.exp(s - m)
            total = p.sum(-1, keepdim=True)
            out[row + a:row + b] = ((p @ v) / total).permute(2, 0, 1, 3).reshape(b - a, heads, d).to(q.dtype)
            lse[row + a:row + b] = (m + torch.log(total)).squeeze(-1).permute(2, 0, 1).reshape(b - a, heads)
        row += n
    return [out, lse]


def _plain_words(refs):
    free = torch.nn.functional.pad((refs == 0).long(), (0, -refs.numel() % 32)).view(-1, 32)
    return (free << torch.arange(32, device=refs.device)).sum(1).to(torch.int32)


def _plain_append(state):
    """The pages that a sequence lacks are the lowest free ones, in the order of the sequences and their tokens."""
    case, ps, cache = state["case"], state["case"]["page"], _split(state["meta"], state["seqs"], state["pages"])
    state["meta"].copy_(state["meta0"])
    old = cache["lengths"].long()
    now = old + state["counts"]
    j = torch.arange(cache["table"].shape[1], device=old.device)
    lacks = ((j * ps < now[:, None]) & (cache["table"] < 0)).view(-1)
    free = torch.argsort((cache["refs"] > 0).to(torch.int8), stable=True)
    got = free[(torch.cumsum(lacks, 0) - 1).clamp(0, state["pages"] - 1)]
    cache["table"].copy_(torch.where(lacks, got.to(torch.int32), cache["table"].reshape(-1)).view_as(cache["table"]))
    cache["refs"].scatter_add_(0, got, lacks.to(torch.int32))
    cache["words"].copy_(_plain_words(cache["refs"]))
    cache["lengths"].copy_(now)
    row = torch.arange(state["k"].shape[0], device=old.device)
    seq = (row[:, None] >= state["starts"][1:]).sum(1)
    pos = old[seq] + row - state["starts"][seq]
    page = cache["table"][seq, pos // ps].long()
    state["pool"][page, 0, 0, :, pos % ps] = state["k"]
    state["pool"][page, 0, 1, :, pos % ps] = state["v"]
    return [state["meta"], state["pool"]]


def _plain_fork(state):
    case, ps, cache = state["case"], state["case"]["page"], _split(state["meta"], state["seqs"], state["pages"])
    state["meta"].copy_(state["meta0"])
    mothers, kids = state["parents"].long(), state["children"].long()
    length = cache["lengths"][mothers].long()
    part = length % ps != 0
    free = torch.argsort((cache["refs"] > 0).to(torch.int8), stable=True)
    fresh = free[(torch.cumsum(part, 0) - 1).clamp_min(0)]
    last = ((length + ps - 1) // ps - 1).clamp_min(0)
    was = cache["table"][mothers, last].long()
    row = cache["table"][mothers]
    row.scatter_(1, last[:, None], torch.where(part, fresh, was).to(torch.int32)[:, None])
    cache["table"][kids] = row
    cache["refs"].scatter_add_(0, row.clamp_min(0).view(-1).long(), (row >= 0).view(-1).to(torch.int32))
    cache["words"].copy_(_plain_words(cache["refs"]))
    cache["lengths"][kids] = length.to(torch.int32)
    to = torch.where(part, fresh, was)
    state["pool"][to] = state["pool"][was]
    return [state["meta"], state["pool"]]


def _plain_retire(state):
    """Pages at or past the number of live ones move, in order, to the free ones below it, in order."""
    cache, pages = _split(state["meta"], state["seqs"], state["pages"]), state["pages"]
    state["meta"].copy_(state["meta0"])
    done = state["done"].long()
    row = cache["table"][done]
    cache["refs"].scatter_add_(0, row.clamp_min(0).view(-1).long(), -(row >= 0).view(-1).to(torch.int32))
    cache["table"][done] = -1
    cache["lengths"][done] = 0
    refs = cache["refs"].clone()
    live = refs > 0
    count, page = live.sum(), torch.arange(pages, device=refs.device)
    moves, hole = live & (page >= count), ~live & (page < count)
    src = torch.argsort((~moves).to(torch.int8), stable=True)[:pages // 2]
    dst = torch.argsort((~hole).to(torch.int8), stable=True)[:pages // 2]
    real = torch.arange(pages // 2, device=refs.device) < moves.sum()
    src = torch.where(real, src, src[0])                  # past the last move: the first one again
    to = torch.where(real, dst, torch.where(real[0], dst[0], src[0]))
    state["pool"][to] = state["pool"][src]
    moved = page.clone()
    moved[src] = to
    cache["refs"].zero_().scatter_add_(0, moved, refs)
    cache["words"].copy_(_plain_words(cache["refs"]))
    table = cache["table"]
    table.copy_(torch.where(table >= 0, moved[table.clamp_min(0).long()].to(torch.int32), table))
    return [state["meta"], state["pool"]]


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(state):
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    from slotstream_b200.kernels import paged_attention
    from slotstream_b200.kv_cache import PagedKvCache
    if "cache" not in state:      # the handle over its tensors, which a program keeps
        state["cache"] = PagedKvCache.over(state["pool"], state["meta"], state["seqs"])
    case, cache = state["case"], state["cache"]
    if case["op"] == "decode":
        q = state["q"]
        lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device)
        o = paged_attention.attn_decode(q, cache.k(0), cache.v(0), cache.table, cache.lengths, lse=lse,
                                        window=case["window"], sinks=case["sinks"])
        return [o, lse]
    if case["op"] == "prompt":
        q = state["q"]
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
        o = paged_attention.attn_prefill(q, cache.k(0), cache.v(0), cache.table, cache.lengths, state["starts"],
                                         lse=lse, window=case["window"], sinks=case["sinks"])
        return [o, lse]
    state["meta"].copy_(state["meta0"])
    if case["op"] == "append":
        cache.extend(state["ids"], state["counts"])
        cache.write(0, state["k"], state["v"], state["starts"])
    elif case["kind"] == "fork":
        cache.fork(state["parents"], state["children"])
    else:
        cache.free(state["done"])
        cache.compact()
    return [state["meta"], state["pool"]]


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    if case["op"] == "decode":
        return _plain_decode(state)
    if case["op"] == "prompt":
        return _plain_prompt(state)
    if case["op"] == "append":
        return _plain_append(state)
    return _plain_fork(state) if case["kind"] == "fork" else _plain_retire(state)


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_attention(state):
    """Every sequence, key head and block of queries by itself: softmax over the tokens that the block can see."""
    case, q = state["case"], state["q"]
    cache = _split(state["meta"], state["seqs"], state["pages"])
    q = q if q.dim() == 3 else q.flatten(0, 1)
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    ps, g = case["page"], case["heads"] // case["kv_heads"]
    lens, row = cache["lengths"].tolist(), 0
    for i in range(case["seqs"]):
        n = case.get("q_len") or state["new"][i]
        for a in range(0, n, 512):
            pos = torch.arange(lens[i] - n + a, lens[i] - n + min(a + 512, n), device=q.device)
            rows = row + a + torch.arange(pos.numel(), device=q.device)
            top = int(pos[-1])
            t = torch.arange(0, max(top + 1, 0), device=q.device)
            if case["window"]:
                t = t[(t > int(pos[0]) - case["window"]) | (t < case["sinks"])]
            if not t.numel():
                continue
            hidden = t[None] > pos[:, None]
            if case["window"]:
                hidden |= (t[None] <= pos[:, None] - case["window"]) & (t[None] >= case["sinks"])
            where = cache["table"][i, t // ps].long() * ps + t % ps
            for h in range(case["kv_heads"]):
                flat = state["pool"][:, 0, :, h].transpose(0, 1)
                k = flat[0, where // ps, where % ps].double()
                v = flat[1, where // ps, where % ps].double()
                x = q[rows, h * g:(h + 1) * g].double()                                   # [R, g, d]
                s = torch.einsum("rgd,td->rgt", x, k).div_(math.sqrt(case["dim"]))
                s.masked_fill_(hidden[:, None], -math.inf)
                z = torch.logsumexp(s, -1)
                w = torch.exp(s - z[..., None]).nan_to_num_(0.0)
                o[rows, h * g:(h + 1) * g] = torch.einsum("rgt,td->rgd", w, v)
                lse[rows, h * g:(h + 1) * g] = z
        row += n
    return [o.view(state["q"].shape), lse.view(state["q"].shape[:-1])]


def _exact_pages(state):
    """The cache's rules on the host, page by page; the data as a list of copies."""
    case, ps, pages, n = state["case"], state["case"]["page"], state["pages"], state["seqs"]
    flat = state["meta0"].cpu()
    c = {k: v.numpy().copy() for k, v in _split(flat, n, pages).items()}
    lens, refs, table, pool = c["lengths"], c["refs"], c["table"], state["pool"].clone()

    def take():
        p = int(np.flatnonzero(refs == 0)[0])
        refs[p] = 1
        return p

    copies = []
    if case["op"] == "append":
        row = 0
        for i, new in enumerate(state["new"]):
            begin = int(lens[i])
            lens[i] += new
            for j in range(-(-int(lens[i]) // ps)):
                if table[i, j] < 0:
                    table[i, j] = take()
            pos = np.arange(begin, begin + new)
            to = torch.from_numpy(table[i, pos // ps].astype(np.int64)).cuda()
            slot = torch.from_numpy(pos % ps).cuda()
            pool[to, 0, 0, :, slot] = state["k"][row:row + new]
            pool[to, 0, 1, :, slot] = state["v"][row:row + new]
            row += new
    elif case["kind"] == "fork":
        for m, k in zip(state["parents"].tolist(), state["children"].tolist()):
            lens[k] = lens[m]
            for j in range(-(-int(lens[m]) // ps)):
                p = int(table[m, j])
                if (j + 1) * ps > lens[m]:
                    table[k, j] = take()
                    copies.append((p, int(table[k, j])))
                else:
                    table[k, j] = p
                    refs[p] += 1
    else:
        for i in state["done"].tolist():
            for j in np.flatnonzero(table[i] >= 0):
                refs[table[i, j]] -= 1
            table[i], lens[i] = -1, 0
        live = np.flatnonzero(refs > 0)
        holes = [p for p in range(live.size) if refs[p] == 0]
        copies = list(zip([int(p) for p in live if p >= live.size], holes))
        for src, dst in copies:
            table[table == src] = dst
            refs[dst], refs[src] = refs[src], 0
    for src, dst in copies:
        pool[dst] = state["pool"][src]
    meta = np.concatenate([lens, refs, _words(refs == 0), table.reshape(-1), c["err"]])
    return [torch.from_numpy(meta).cuda(), pool]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] in ("decode", "prompt"):
        return _exact_attention(state)
    return _exact_pages(state)
