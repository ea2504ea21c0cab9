"""Plain 64-bit forms of the paged-cache operators: a host model of the page rules, and attention by its definition
with an element-wise error bound derived from the roundings that the kernels are allowed."""
import math

import numpy as np
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # half an ulp, relative


class CacheModel:
    """The rules of the paged cache on the host: lengths, refs and table as numpy arrays, pages as numbers only;
    ``copies`` lists the (source, target) pages whose data a call moves."""

    def __init__(self, pages, page_size, seqs, max_pages):
        self.ps, self.pages, self.max_pages = page_size, pages, max_pages
        self.lengths = np.zeros(seqs, np.int32)
        self.refs = np.zeros(pages, np.int32)
        self.table = np.full((seqs, max_pages), -1, np.int32)
        self.copies = []

    def held(self, s):
        return -(-int(self.lengths[s]) // self.ps)

    def extend(self, ids, counts):
        lens = self.lengths.copy()
        want = []
        for s, n in zip(ids, counts):
            lens[s] += n
            if n:
                want += [(s, j) for j in range(int(self.lengths[s]) // self.ps, -(-int(lens[s]) // self.ps))
                         if self.table[s, j] < 0]
        free = np.flatnonzero(self.refs == 0)
        assert len(want) <= free.size
        for (s, j), p in zip(want, free):
            self.table[s, j], self.refs[p] = p, 1
        self.lengths = lens

    def fork(self, parents, children):
        free = list(np.flatnonzero(self.refs == 0))
        before = self.lengths.copy()
        for p, c in zip(parents, children):
            n = int(before[p])
            for j in range(n // self.ps):
                page = self.table[p, j]
                self.table[c, j] = page
                if page >= 0:
                    self.refs[page] += 1
            if n % self.ps and self.table[p, n // self.ps] >= 0:
                fresh = free.pop(0)
                self.copies.append((int(self.table[p, n // self.ps]), int(fresh)))
                self.table[c, n // self.ps], self.refs[fresh] = fresh, 1
            self.lengths[c] = n

    def free(self, ids, first=None, last=None):
        for i, s in enumerate(ids):
            for j in range(self.max_pages) if first is None else range(max(first[i], 0), min(last[i], self.max_pages)):
                if self.table[s, j] >= 0:
                    self.refs[self.table[s, j]] -= 1
                    self.table[s, j] = -1
            if first is None:
                self.lengths[s] = 0

    def release(self, ids, first, last):
        self.free(ids, first, last)

    def compact(self):
        live = int((self.refs > 0).sum())
        src = [p for p in range(live, self.pages) if self.refs[p]]
        dst = [p for p in range(live) if not self.refs[p]]
        for s, d in zip(src, dst):
            self.copies.append((s, d))
            self.table[self.table == s] = d
            self.refs[d], self.refs[s] = self.refs[s], 0

    def words(self):
        bits = np.zeros(-(-self.pages // 32) * 32, np.int64)
        bits[:self.pages] = self.refs == 0
        return (bits.reshape(-1, 32) << np.arange(32)).sum(1).astype(np.uint32).view(np.int32)

    def state(self):
        return np.concatenate([self.lengths, self.refs, self.words(), self.table.reshape(-1), np.zeros(1, np.int32)])


def attention(q, k_pages, v_pages, table, lengths, q_lens, window=0, sinks=0, scale=None, ids=None):
    """q [rows, heads, dim], the q_lens[b] rows of sequence b after one another. Returns o, lse (64 bits) and the bounds
    of a kernel's error in each: the weights and the result rounded to the type (u each), scores summed in fp32 by the
    tensor cores (dim terms, 2^-22 each, of the sum of magnitudes), everything else in fp32 (2^-18 of the magnitudes)."""
    rows, heads, dim = q.shape
    kv, ps = k_pages.shape[1], k_pages.shape[2]
    g, u = heads // kv, UNIT[q.dtype]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    o = torch.zeros(rows, heads, dim, dtype=torch.float64, device=q.device)
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64, device=q.device)
    o_tol, lse_tol = torch.zeros_like(o), torch.zeros_like(lse)
    tab, lens, row = table.cpu().numpy(), lengths.cpu().numpy(), 0
    for b, n in enumerate(q_lens):
        s = b if ids is None else int(ids[b])
        length = int(lens[s])
        for i in range(n):
            p = length - n + i
            t = np.arange(max(p + 1, 0))
            if window:
                t = t[(p - t < window) | (t < sinks)]
            if t.size:
                page = torch.from_numpy(tab[s, t // ps].astype(np.int64)).to(q.device)
                slot = torch.from_numpy(t % ps).to(q.device)
                k = k_pages[page, :, slot].double().transpose(0, 1)              # [kv, T, D]
                v = v_pages[page, :, slot].double().transpose(0, 1)
                x = q[row + i].double().view(kv, g, dim)
                score = (x @ k.transpose(1, 2)) * scale
                size = (x.abs() @ k.abs().transpose(1, 2)).amax(-1) * abs(scale) * dim * 2.0 ** -22   # [kv, g]
                z = torch.logsumexp(score, -1)
                w = torch.exp(score - z[..., None])
                res, mass = w @ v, w @ v.abs()
                o[row + i], lse[row + i] = res.reshape(heads, dim), z.reshape(heads)
                tol = u * res.abs() + (u + 2 * size[..., None] + 2.0 ** -18) * mass * 1.01
                o_tol[row + i] = tol.reshape(heads, dim) + 1e-7
                lse_tol[row + i] = (size + 2.0 ** -20 * (1 + z.abs()) + 2.0 ** -18).reshape(heads)
        row += n
    return o, lse, o_tol, lse_tol


def assert_attention(out, lse, ref):
    o, z, o_tol, z_tol = ref
    bad = (out.double() - o).abs() > o_tol
    assert not bool(bad.any()), f"{int(bad.sum())} outputs past their bound, worst {float((out.double() - o).abs().max())}"
    assert not bool(torch.isnan(out).any())
    assert bool((torch.isneginf(lse) == torch.isneginf(z)).all())
    fine = ~torch.isneginf(z)
    assert bool(((lse.double() - z).abs()[fine] <= z_tol[fine]).all())
