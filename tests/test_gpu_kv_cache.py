"""Paged key-value cache against a host model of its rules (GPU): whole state and data after every call."""
import numpy as np
import pytest
import torch

from paged_reference import CacheModel
from slotstream_b200.kv_cache import PagedKvCache

pytestmark = pytest.mark.gpu


def _t(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


class Pair:
    """A cache and its model, compared after every call; page data are told apart by random contents."""

    def __init__(self, pages=37, layers=2, kv=2, ps=4, dim=8, seqs=9, max_pages=6, dtype=torch.bfloat16):
        self.c = PagedKvCache(pages, layers, kv, ps, dim, seqs, max_pages, dtype)
        self.c.pool.copy_(torch.randn(self.c.pool.shape, device="cuda"))
        self.m = CacheModel(pages, ps, seqs, max_pages)

    def check(self):
        torch.cuda.synchronize()
        got = self.c.state.cpu().numpy()
        assert np.array_equal(got, self.m.state())

    def call(self, name, *args):
        before = self.c.pool.clone()
        self.m.copies = []
        getattr(self.c, name)(*[_t(a) for a in args])
        getattr(self.m, name)(*args)
        self.check()
        for s, d in self.m.copies:
            before[d] = before[s]
        assert torch.equal(self.c.pool, before)

    def refused(self, bit, name, *args):
        state, pool = self.c.state.clone(), self.c.pool.clone()
        getattr(self.c, name)(*[_t(a) for a in args])
        torch.cuda.synchronize()
        assert int(self.c.err.item()) == bit
        with pytest.raises(RuntimeError, match="kv cache"):
            self.c.check()
        self.c.check()                                  # cleared
        assert torch.equal(self.c.state, state) and torch.equal(self.c.pool, pool)


def test_new_cache_is_empty():
    for pages in (1, 31, 32, 33, 64):
        Pair(pages=pages).check()


def test_life_of_sequences():
    p = Pair()
    p.call("extend", [0, 3, 1], [5, 4, 1])
    p.call("extend", [3, 0], [1, 0])
    p.call("fork", [0, 3, 0], [5, 6, 8])
    p.call("extend", [5, 0, 6, 8], [3, 4, 1, 9])
    p.call("free", [0, 1])
    p.call("compact")
    p.call("extend", [1, 0, 2], [24, 3, 11])
    p.call("release", [1], [1], [3])
    p.call("release", [1, 8], [-4, 1], [2, 99])
    p.call("compact")
    p.call("free", [1, 2, 3, 5, 6, 8, 0, 0])
    p.call("compact")
    assert int(p.m.refs.sum()) == 0


@pytest.mark.parametrize("seed", range(6))
def test_random_lives(seed):
    """Random calls on caches whose pages end at, before and past a word of free bits."""
    r = np.random.default_rng(seed)
    p = Pair(pages=int(r.integers(20, 140)), ps=int(r.integers(1, 9)), seqs=12, max_pages=8, layers=int(r.integers(1, 3)))
    m = p.m
    for _ in range(25):
        live, empty = np.flatnonzero(m.lengths > 0), np.flatnonzero(m.lengths == 0)
        what = r.choice(["extend", "fork", "free", "compact"])
        if what == "extend":
            ids = r.permutation(12)[:r.integers(1, 13)]
            counts = [int(min(r.integers(0, 2 * m.ps + 2), 8 * m.ps - m.lengths[s])) for s in ids]
            need = sum(-(-(m.lengths[s] + n) // m.ps) - m.held(s) for s, n in zip(ids, counts))
            if need <= int((m.refs == 0).sum()):
                p.call("extend", ids.tolist(), counts)
        elif what == "fork" and live.size and empty.size:
            kids = r.permutation(empty)[:r.integers(1, empty.size + 1)].tolist()
            mothers = r.choice(live, len(kids)).tolist()
            if len(kids) <= int((m.refs == 0).sum()):
                p.call("fork", mothers, kids)
        elif what == "free" and live.size:
            p.call("free", r.permutation(live)[:r.integers(1, live.size + 1)].tolist())
        elif what == "compact":
            p.call("compact")


def test_many_pages_and_sequences():
    """Free words of several per thread, more sequences than a plan has warps and threads."""
    p = Pair(pages=70000, layers=1, kv=1, ps=2, dim=8, seqs=1500, max_pages=60)
    ids = np.random.default_rng(0).permutation(1500).tolist()
    p.call("extend", ids[:1400], [int(i % 90) for i in range(1400)])
    p.call("fork", ids[:80], ids[1400:1480])
    p.call("free", ids[:700])
    p.call("compact")
    p.call("extend", ids[:700], [60] * 700)


def test_large_pages():
    """Pages that end inside a copy piece."""
    p = Pair(pages=20, layers=3, kv=3, ps=24, dim=128, seqs=6, max_pages=4)
    p.call("extend", [0, 1, 2], [30, 50, 24])
    p.call("fork", [0, 1, 2], [3, 4, 5])
    p.call("free", [0, 1])
    p.call("compact")


def test_refusals_on_the_device_change_nothing():
    p = Pair(pages=8, ps=4, seqs=6, max_pages=4)
    p.call("extend", [0, 1], [6, 8])
    p.refused(32, "extend", [2, 3], [9, 9])             # too few pages
    p.refused(32, "extend", [0], [11])                  # past the table row
    p.refused(64, "extend", [2, 2], [1, 1])
    p.refused(64, "extend", [6], [1])
    p.refused(64, "extend", [-1], [1])
    p.refused(64, "extend", [2], [-1])
    p.refused(64, "fork", [0], [1])                     # the child holds tokens
    p.refused(64, "fork", [0, 0], [2, 2])
    p.refused(64, "fork", [0], [6])
    p.refused(64, "fork", [-1], [2])
    p.call("fork", [1], [2])
    p.c.lengths[2] -= 2                                 # rolled back into a shared page
    p.refused(256, "extend", [2], [1])
    p.c.lengths[2] += 2
    p.call("extend", [3], [16])
    p.refused(32, "fork", [0], [4])                     # no page for the copy of the partial one
    p.c.free(_t([9]))
    with pytest.raises(RuntimeError, match="sequence id"):
        p.c.check()


def test_fork_of_a_child_of_the_same_call_copies_what_was_there():
    p = Pair()
    p.call("extend", [0], [7])
    p.call("fork", [0, 1, 1], [1, 2, 3])                # sequence 1 is empty when the call begins


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kv,dim,ps", [(1, 8, 1), (2, 64, 16), (3, 40, 7), (8, 128, 32)])
def test_write(dtype, kv, dim, ps):
    """Rows of strided projections land in their slots, nothing else changes."""
    c = PagedKvCache(64, 2, kv, ps, dim, 5, 40, dtype)
    c.pool.copy_(torch.randn(c.pool.shape, device="cuda"))
    c.extend(_t([0, 1, 2, 3, 4]), _t([3, 0, 7, 1, 2]))
    new = [4, 0, 1, ps]
    ids = [4, 1, 0, 2]
    c.extend(_t(ids), _t(new))
    c.check()
    both = torch.randn(sum(new) + 2, 3 * kv, dim, device="cuda").to(dtype)
    k, v = both[:, :kv], both[:, 2 * kv:]
    want = c.pool.clone()
    table, lens, row = c.table.cpu().numpy(), c.lengths.cpu().numpy(), 0
    for s, n in zip(ids, new):
        for i in range(n):
            t = lens[s] - n + i
            want[table[s, t // ps], 1, 0, :, t % ps] = k[row]
            want[table[s, t // ps], 1, 1, :, t % ps] = v[row]
            row += 1
    c.write(1, k, v, _t(np.cumsum([0] + new)), _t(ids))   # two rows past the last sequence: not written
    c.check()
    assert torch.equal(c.pool, want)


def test_write_refuses_shared_and_missing_pages():
    c = PagedKvCache(16, 1, 1, 4, 8, 4, 4)
    c.pool.zero_()
    c.extend(_t([0]), _t([8]))
    c.fork(_t([0]), _t([1]))
    c.check()
    k = torch.ones(1, 1, 8, dtype=torch.bfloat16, device="cuda")
    for ids, message in ((1, "another sequence"), (7, "sequence id"), (2, "sequence id")):
        c.write(0, k, k, _t([0, 1]), _t([ids]))
        with pytest.raises(RuntimeError, match=message):
            c.check()
    c.lengths[1] += 1                                     # a token without a page
    c.write(0, k, k, _t([0, 1]), _t([1]))
    with pytest.raises(RuntimeError, match="missing page"):
        c.check()
    assert not bool(c.pool.any())


def test_calls_can_be_captured():
    p = Pair()
    p.call("extend", [0, 1], [6, 6])
    ids, counts = _t([0, 1]), _t([1, 1])
    k = torch.randn(2, 2, 8, device="cuda").to(torch.bfloat16)
    starts = _t([0, 1, 2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.c.extend(ids, counts)
        p.c.write(0, k, k, starts)
    for _ in range(5):
        graph.replay()
        p.m.extend([0, 1], [1, 1])
        p.check()
        for s in (0, 1):
            t = int(p.m.lengths[s]) - 1
            assert torch.equal(p.c.k(0)[int(p.m.table[s, t // 4]), :, t % 4], k[s])
