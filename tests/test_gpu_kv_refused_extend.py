"""Writes after an extend that was refused: the tokens that are cached stay as they are, and a retry is right (GPU)."""
import pytest
import torch

from slotstream_b200.kv_cache import PagedKvCache

pytestmark = pytest.mark.gpu


def _t(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def _rows(n, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(n, 2, 8, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2)]


def _full(seqs=4, pages=6):
    """Sequences 0 and 1 of 8 and 6 tokens and sequence 2 of 5, pages of 4 tokens, of which they hold six; data written."""
    c = PagedKvCache(pages, 2, 2, 4, 8, seqs, 4)
    c.pool.zero_()
    c.extend(_t([0, 1, 2]), _t([8, 6, 5]))
    for layer in range(2):
        c.write(layer, *_rows(19, layer), _t([0, 8, 14, 19]))
    c.check()
    assert bool(c.pool.any()) and int((c.refs == 0).sum()) == pages - 6
    return c


def _step(c, ids, counts, seed=9):
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + max(n, 0))
    rows = [_rows(max(starts[-1], 1), seed + layer) for layer in range(2)]
    c.extend(_t(ids), _t(counts))
    for layer in range(2):
        c.write(layer, *rows[layer], _t(starts), _t(ids))
    return rows


@pytest.mark.parametrize("ids,counts,match", [
    ([0, 1], [1, 1], "not enough free pages"),               # sequence 0 needs a page and there is none
    ([1, 0], [2, 9], "not enough free pages"),               # past the table row
    ([1, 1], [1, 1], "sequence id"),
    ([1, 9], [1, 1], "sequence id"),
    ([1, 0], [1, -1], "sequence id"),
])
def test_a_write_after_a_refused_extend_changes_nothing(ids, counts, match):
    c = _full()
    pool, lengths, table = c.pool.clone(), c.lengths.clone(), c.table.clone()
    _step(c, ids, counts)
    assert torch.equal(c.pool, pool) and torch.equal(c.lengths, lengths) and torch.equal(c.table, table)
    with pytest.raises(RuntimeError, match=match):
        c.check()
    c.write(0, *_rows(1, 5), _t([0, 1]), _t([1]))            # the error was read; there is still no room for the row
    with pytest.raises(RuntimeError, match="refused"):
        c.check()
    assert torch.equal(c.pool, pool)


def test_a_write_after_an_extend_into_a_shared_page_changes_nothing():
    c = _full(pages=9)                      # three more pages, which sequences 3 and its kin take
    c.extend(_t([3]), _t([8]))
    c.free(_t([2]))
    c.fork(_t([3]), _t([2]))
    c.check()
    c.lengths[2] -= 2                       # rolled back into a shared page
    pool = c.pool.clone()
    _step(c, [1, 2], [1, 1])
    assert torch.equal(c.pool, pool)
    with pytest.raises(RuntimeError, match="another sequence"):
        c.check()


def test_a_retry_after_pages_were_freed_is_right_and_others_go_on():
    c = _full()
    pool = c.pool.clone()
    _step(c, [0, 1], [1, 1])
    assert torch.equal(c.pool, pool)
    with pytest.raises(RuntimeError):
        c.check()
    (k, v), _ = _step(c, [2], [1], seed=30)                  # sequence 2 was not named and has room
    c.check()
    page, slot = int(c.table[2, 1]), 1
    assert torch.equal(c.k(0)[page, :, slot], k[0]) and torch.equal(c.v(0)[page, :, slot], v[0])
    c.free(_t([2]))
    pool.copy_(c.pool)
    rows = _step(c, [0, 1], [1, 1], seed=50)
    c.check()
    assert c.lengths.tolist() == [9, 7, 0, 0]
    for s, t, row in ((0, 8, 0), (1, 6, 1)):
        page = int(c.table[s, t // 4])
        for layer, (k, v) in enumerate(rows):
            pool[page, layer, 0, :, t % 4], pool[page, layer, 1, :, t % 4] = k[row], v[row]
    assert torch.equal(c.pool, pool)


def test_a_captured_step_that_is_refused_once():
    c = _full()
    ids, counts, starts, rows = _t([0, 1]), _t([1, 1]), _t([0, 1, 2]), _rows(2, 3)
    done, graph, state = _t([2]), torch.cuda.CUDAGraph(), c.state.clone()
    with torch.cuda.graph(graph):
        c.extend(ids, counts)
        c.write(1, *rows, starts, ids)
    assert torch.equal(c.state, state)
    pool = c.pool.clone()
    graph.replay()
    assert torch.equal(c.pool, pool)
    c.free(done)                                              # nobody has looked at the error yet
    graph.replay()
    for s, t in ((0, 8), (1, 6)):
        page = int(c.table[s, t // 4])
        pool[page, 1, 0, :, t % 4], pool[page, 1, 1, :, t % 4] = rows[0][s], rows[1][s]
    assert torch.equal(c.pool, pool) and c.lengths.tolist() == [9, 7, 0, 0]


def test_a_sequence_that_asked_for_nothing_can_still_be_written():
    c = _full()
    c.extend(_t([1]), _t([1]))
    c.extend(_t([1, 0]), _t([0, 1]))                          # no page for sequence 0
    k, v = _rows(1, 4)
    c.write(0, k, v, _t([0, 1]), _t([1]))
    with pytest.raises(RuntimeError, match=r"not enough free pages.*\(error bits 32\)"):
        c.check()
    assert torch.equal(c.k(0)[int(c.table[1, 1]), :, 2], k[0])


def test_more_sequences_than_a_block_has_threads():
    n = 1500
    c = PagedKvCache(n, 1, 2, 2, 8, n, 2)
    c.pool.zero_()
    ids = torch.randperm(n, device="cuda").to(torch.int32)
    one, starts = torch.ones_like(ids), torch.arange(n + 1, dtype=torch.int32, device="cuda")
    c.extend(ids, one * 2)
    c.check()
    k, v = _rows(n, 1)
    c.extend(ids, one)
    c.write(0, k, v, starts, ids)
    assert not bool(c.pool.any())
    with pytest.raises(RuntimeError, match="not enough free pages"):
        c.check()
