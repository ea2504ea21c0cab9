"""Paged key-value cache for the attention between the MoE layers (additive), over the C entry points ssb_kv_*.

The reference keeps its attention and its cache outside the path that this package replaces; ``PagedKvCache`` gives a
program that runs the MoE layers here a cache for the layers between them. Keys and values of ``page_size`` consecutive
tokens, of every layer, form one page of ``pool`` [pages, layers, 2, kv_heads, page_size, head_dim] (so a page is one
contiguous run of bytes to copy, and ``k(layer)`` / ``v(layer)`` are strided views for ``kernels.paged_attention``);
``table`` [seqs, max_pages] names each sequence's pages, -1 where it has none.

All state is device memory and every call only launches on the current stream: nothing waits for the host, and the calls
can be captured in a CUDA graph. What the device finds wrong -- no free pages, a bad or repeated sequence, a shared page
about to be written -- sets a bit in ``err``; ``check()`` reads it (and waits for it). ``extend`` and ``fork`` then leave the
state as it was; ``free`` and ``release`` pass over bad ids, and ``write`` drops the rows that have no place. After an
``extend`` that was refused, ``write`` drops the rows of the sequences that it was to give room, until an ``extend`` has made
it, so that a step need not look in between; the attention of that step sees the tokens of before. Which sequences wait for
room is kept in ``scratch``, so calls that belong together go through one ``PagedKvCache``.

A decode step: ``extend(ids, counts)`` once (lengths grow, pages are allocated), then per layer ``write(layer, k, v,
starts, ids)``, ``attn_decode(q, cache.k(layer), cache.v(layer), cache.table, cache.lengths, ids=ids)`` and the MoE layer.
"""
import ctypes

import torch

from . import _lib

_TYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_ERRORS = {_lib.ERR_NO_PAGES: "not enough free pages, or a table row is full",
           _lib.ERR_SEQUENCE: "a sequence id out of range or repeated, a bad count, or a fork onto a held sequence",
           _lib.ERR_PAGE_RANGE: "a missing page or one outside the pool",
           _lib.ERR_SHARED_PAGE: "new tokens in a page that another sequence holds too",
           _lib.ERR_NO_ROOM: "rows for a sequence whose last extend was refused, which were dropped",
           _lib.ERR_TIMEOUT: "a wait inside a prompt's attention gave up, and rows of its output were not written",
           _lib.ERR_MISALIGNED: "the prompt attention kernel's shared memory was not aligned, and no output was written"}


def state_ints(pages: int, seqs: int, max_pages: int) -> int:
    """int32 words of the cache's state: lengths, refs, free words, table, error word, in this order."""
    return seqs + pages + (pages + 31) // 32 + seqs * max_pages + 1


def _ids(t, name, n=None):
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() or (n is not None and t.numel() != n):
        raise ValueError(f"{name} must be a contiguous int32 vector" + (f" of {n}" if n is not None else ""))
    return _lib.ptr(t)


class PagedKvCache:
    def __init__(self, pages: int, layers: int, kv_heads: int, page_size: int, head_dim: int, seqs: int,
                 max_pages: int, dtype=torch.bfloat16, device="cuda"):
        if min(pages, layers, kv_heads, page_size, head_dim, seqs, max_pages) < 1:
            raise ValueError("every size of a cache is at least 1")
        pool = torch.empty(pages, layers, 2, kv_heads, page_size, head_dim, dtype=dtype, device=device)
        state = torch.zeros(state_ints(pages, seqs, max_pages), dtype=torch.int32, device=device)
        self._bind(pool, state, seqs)
        self.reset()

    @classmethod
    def over(cls, pool, state, seqs: int):
        """A cache over tensors that the caller holds: ``pool`` as above and ``state`` (int32, ``state_ints`` words),
        whose contents are taken as they are."""
        c = cls.__new__(cls)
        c._bind(pool, state, seqs)
        return c

    def _bind(self, pool, state, seqs):
        if pool.dim() != 6 or pool.shape[2] != 2 or not pool.is_contiguous() or pool.dtype not in _TYPES:
            raise ValueError("pool must be a contiguous bf16 or fp16 [pages, layers, 2, kv_heads, page_size, head_dim]")
        self.pages, self.layers, _, self.kv_heads, self.page_size, self.head_dim = pool.shape
        if self.head_dim % 8:
            raise ValueError(f"head_dim must be a multiple of 8, got {self.head_dim}")
        words = (self.pages + 31) // 32
        rest = state.numel() - 1 - seqs - self.pages - words
        if state.dtype != torch.int32 or state.dim() != 1 or not state.is_contiguous() or seqs < 1 or rest < seqs \
                or rest % seqs:
            raise ValueError("state must be a contiguous int32 vector of state_ints(pages, seqs, max_pages)")
        self.pool, self.state, self.seqs, self.max_pages = pool, state, seqs, rest // seqs
        o = [0, seqs, seqs + self.pages, seqs + self.pages + words, state.numel() - 1]
        self.lengths, self.refs, self.free_words = state[:o[1]], state[o[1]:o[2]], state[o[2]:o[3]]
        self.table, self.err = state[o[3]:o[4]].view(seqs, self.max_pages), state[o[4]:]
        L = _lib.lib()
        ints = L.ssb_kv_scratch_ints(self.pages, seqs)
        if ints < 0:
            raise ValueError(f"a cache has at most 2^20 pages and 65536 sequences, got {self.pages} and {seqs}")
        self.scratch = torch.zeros(ints, dtype=torch.int32, device=pool.device)
        p = _lib.ptr
        self._struct = _lib.KvCacheStruct(p(pool), pool[0].numel() * pool.element_size(), self.pages, self.page_size, seqs,
                                          self.max_pages, p(self.lengths), p(self.refs), p(self.free_words),
                                          p(self.table), p(self.err), p(self.scratch))
        self._c = ctypes.addressof(self._struct)
        self._k = [pool[:, i, 0] for i in range(self.layers)]
        self._v = [pool[:, i, 1] for i in range(self.layers)]
        self._strides = self._k[0].stride()

    def reset(self):
        """Every sequence empty, every page free, no error."""
        self.state.zero_()
        self.scratch.zero_()
        self.table.fill_(-1)
        self.free_words.fill_(-1)
        if self.pages % 32:
            self.free_words[-1:].fill_((1 << (self.pages % 32)) - 1)

    def k(self, layer: int):
        """Keys of a layer: [pages, kv_heads, page_size, head_dim], a view of the pool."""
        return self._k[layer]

    def v(self, layer: int):
        return self._v[layer]

    def extend(self, ids, counts):
        """lengths[ids[i]] += counts[i] (int32 vectors on the device), with the lowest free pages for the new tokens; all of
        them or, when something is wrong, none."""
        n = ids.numel()
        if n > self.seqs:
            raise ValueError(f"{n} sequences named, the cache has {self.seqs}")
        rc = _lib.lib().ssb_kv_extend(self._c, _ids(ids, "ids"), _ids(counts, "counts", n), n, _lib.stream())
        _lib.check(rc, "kv extend")

    def write(self, layer: int, k, v, starts, ids=None):
        """Keys and values [rows, kv_heads, head_dim] of the newest tokens into one layer. Rows ``starts[b]`` to
        ``starts[b + 1]`` (int32, on the device) are the newest tokens of sequence ``ids[b]`` (default b), which
        ``extend`` has made room for. The head dimension is contiguous; the other strides are multiples of 8."""
        if k.dtype != self.pool.dtype or v.dtype != self.pool.dtype or k.dim() != 3 or k.shape != v.shape \
                or tuple(k.shape[1:]) != (self.kv_heads, self.head_dim):
            raise ValueError(f"k and v must be {self.pool.dtype} [rows, {self.kv_heads}, {self.head_dim}]")
        ks, vs = k.stride(), v.stride()
        if ks[2] != 1 or vs[2] != 1:
            raise ValueError("the head dimension of k and v must be contiguous")
        n = starts.numel() - 1
        if n < 0:
            raise ValueError("starts needs at least one element")
        p, st = _lib.ptr, self._strides
        rows = _lib.KV_ROWS.pack(p(k), p(v), ks[0], ks[1], vs[0], vs[1], k.shape[0], _ids(starts, "starts"),
                                 0 if ids is None else _ids(ids, "ids", n), self._k[layer].data_ptr(),
                                 self._v[layer].data_ptr(), st[0], st[1], st[2], n, self.kv_heads, self.head_dim)
        rc = _lib.lib().ssb_kv_write(self._c, rows, _lib.stream())
        _lib.check(rc, "kv write")

    def fork(self, parents, children):
        """children[i] becomes a copy of parents[i]: full pages are shared, a partly filled last page is copied."""
        n = parents.numel()
        if n > self.seqs:
            raise ValueError(f"{n} sequences named, the cache has {self.seqs}")
        rc = _lib.lib().ssb_kv_fork(self._c, _ids(parents, "parents"), _ids(children, "children", n), n, _lib.stream())
        _lib.check(rc, "kv fork")

    def free(self, ids):
        """Empties the sequences: their pages lose a reference and become free with the last one."""
        rc = _lib.lib().ssb_kv_free(self._c, _ids(ids, "ids"), None, None, ids.numel(), _lib.stream())
        _lib.check(rc, "kv free")

    def release(self, ids, first, last):
        """Gives back pages first[i] to last[i] (exclusive) of the sequences, whose lengths stay: pages that a sliding
        window has passed. Attention must not see them again."""
        n = ids.numel()
        rc = _lib.lib().ssb_kv_free(self._c, _ids(ids, "ids"), _ids(first, "first", n), _ids(last, "last", n), n,
                                    _lib.stream())
        _lib.check(rc, "kv release")

    def compact(self):
        """Moves the live pages to the front of the pool (tables follow): afterwards the free pages are its end."""
        _lib.check(_lib.lib().ssb_kv_compact(self._c, _lib.stream()), "kv compact")

    def check(self):
        """Raises if an error bit is set, and clears it. Waits for the device."""
        bits = int(self.err.item())
        if bits:
            self.err.zero_()
            known = [m for b, m in _ERRORS.items() if bits & b]
            if bits & ~sum(_ERRORS):
                known.append("an unknown error")
            raise RuntimeError("kv cache: " + "; ".join(known) + f" (error bits {bits})")
