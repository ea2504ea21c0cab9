"""Forks onto a sequence of length 0 that still holds pages are refused where its name for one would be lost (GPU)."""
import pytest
import torch

from slotstream_b200.kv_cache import PagedKvCache

pytestmark = pytest.mark.gpu


def _t(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("max_pages", [6, 40, 300, 5000])
@pytest.mark.parametrize("first_kept", [1, 3])
def test_a_child_whose_first_pages_were_released(max_pages, first_kept):
    c = PagedKvCache(64, 1, 1, 4, 8, 8, max_pages)
    c.pool.copy_(torch.randn(c.pool.shape, device="cuda"))
    c.extend(_t([0, 1]), _t([22, 23]))
    c.release(_t([1]), _t([0]), _t([first_kept]))
    c.lengths[1] = 0                                        # rolled back, its later pages still held
    c.check()
    state, pool = c.state.clone(), c.pool.clone()
    c.fork(_t([0, 0, 0]), _t([2, 1, 3]))
    with pytest.raises(RuntimeError, match="held sequence"):
        c.check()
    assert torch.equal(c.state, state) and torch.equal(c.pool, pool)
    c.free(_t([1]))
    c.fork(_t([0, 0, 0]), _t([2, 1, 3]))
    c.check()
    assert c.lengths.tolist()[:4] == [22] * 4
    c.free(_t([0, 1, 2, 3]))
    c.check()
    assert int(c.refs.sum()) == 0 and int(c.table.max()) == -1      # no page has lost its last name


@pytest.mark.parametrize("held", [0, 1, 31, 32, 127, 128, 299, 300])
def test_a_page_anywhere_among_the_entries_that_the_child_gets(held):
    """The parent stands in 301 pages; one of 129 children holds one page, at entry ``held``."""
    c = PagedKvCache(2000, 1, 1, 4, 8, 130, 310)
    c.extend(_t([0]), _t([1201]))
    c.lengths[77] = held * 4                                # as a window would leave it: only this page is there
    c.extend(_t([77]), _t([1]))
    c.lengths[77] = 0
    c.check()
    state, kids = c.state.clone(), [i for i in range(130) if i]
    c.fork(_t([0] * 129), _t(kids))
    with pytest.raises(RuntimeError, match="held sequence"):
        c.check()
    assert torch.equal(c.state, state)


def test_a_page_past_the_entries_that_the_child_gets_stays_its_own():
    c = PagedKvCache(64, 1, 1, 4, 8, 4, 20)
    c.extend(_t([0, 1]), _t([9, 40]))
    c.release(_t([1]), _t([0]), _t([9]))
    page = int(c.table[1, 9])
    c.lengths[1] = 0
    c.fork(_t([0]), _t([1]))
    c.extend(_t([1]), _t([30]))                             # up to token 39: through the page that was kept
    c.check()
    assert int(c.table[1, 9]) == page and int(c.refs[page]) == 1
    c.free(_t([0, 1]))
    c.check()
    assert int(c.refs.sum()) == 0 and int(c.table.max()) == -1
