"""Every error bit that a kernel may set in a cache's error word has a text of its own (CPU)."""
import pytest
import torch

from conftest import ROOT
from slotstream_b200.kv_cache import PagedKvCache


def _bits():
    """SSB_ERR_* of the C header."""
    for line in (ROOT / "include" / "slotstream_b200.h").read_text().splitlines():
        if line.startswith("#define SSB_ERR_"):
            _, name, value = line.split()[:3]
            yield pytest.param(int(value), id=name)


def _message(bits):
    cache = PagedKvCache.__new__(PagedKvCache)
    cache.err = torch.tensor([bits], dtype=torch.int32)
    with pytest.raises(RuntimeError) as e:
        cache.check()
    assert int(cache.err) == 0
    return str(e.value)


USED = {"SSB_ERR_NO_PAGES", "SSB_ERR_SEQUENCE", "SSB_ERR_PAGE_RANGE", "SSB_ERR_SHARED_PAGE", "SSB_ERR_TIMEOUT",
        "SSB_ERR_MISALIGNED"}


@pytest.mark.parametrize("bit", [p for p in _bits() if p.id in USED])
def test_a_text_for_every_bit(bit):
    text = _message(bit).removeprefix("kv cache: ").removesuffix(f" (error bits {bit})")
    assert len(text) > 10


def test_bits_without_a_text_are_named_by_number():
    assert "error bits 1073741824" in _message(1 << 30) and "unknown" in _message(1 << 30)


def test_several_bits():
    assert _message(32 | 16).count(";") == 1
