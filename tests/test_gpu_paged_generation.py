"""The generation loop of examples/paged_generation.py: forks, frees and compaction change nothing that is computed (GPU)."""
import sys

import numpy as np
import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(ROOT / "examples"))


def _copy(cache, parents, children):
    """A fork by hand: every child gets pages of its own, filled from its parent's."""
    cache.extend(children, cache.lengths[parents.long()].contiguous())
    for p, c in zip(parents.tolist(), children.tolist()):
        pages = -(-int(cache.lengths[p]) // cache.page_size)
        cache.pool[cache.table[c, :pages].long()] = cache.pool[cache.table[p, :pages].long()]


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 2)])
def test_shared_pages_give_the_same_tokens_and_logits_as_copies(window, sinks):
    from paged_generation import Model, generate
    r = np.random.default_rng(1)
    prompts = [r.integers(0, 1024, n).tolist() for n in (37, 64, 9)]
    model = Model(window=window, sinks=sinks)
    tokens, logits, cache = generate(model, prompts, samples=2, steps=10)
    want, want_logits, _ = generate(model, prompts, samples=2, steps=10, clone=_copy)
    # the same launches on the same values in other pages: bit for bit
    assert torch.equal(tokens, want) and torch.equal(logits, want_logits)
    assert bool(torch.isfinite(logits).all())
    live = int((cache.refs > 0).sum())
    assert live == int(cache.table.unique().ge(0).sum()) and int(cache.table.max()) < live + 3   # packed, but for new pages


def test_cached_decode_agrees_with_reading_the_whole_sequence_again():
    """One attention layer over the cache against the 64-bit definition, on the loop's own keys and queries."""
    from paged_generation import Model, generate
    from paged_reference import assert_attention, attention
    from slotstream_b200.kernels.paged_attention import attn_decode
    r = np.random.default_rng(2)
    model = Model(layers=1)
    _, _, cache = generate(model, [r.integers(0, 1024, n).tolist() for n in (50, 3)], samples=2, steps=6)
    ids = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 1, model.heads, model.dim, device="cuda").to(torch.bfloat16)
    lse = torch.empty(2, 1, model.heads, device="cuda")
    out = attn_decode(q, cache.k(0), cache.v(0), cache.table, cache.lengths, lse=lse, ids=ids, err=cache.err)
    cache.check()
    assert_attention(out[:, 0], lse[:, 0], attention(q[:, 0], cache.k(0), cache.v(0), cache.table, cache.lengths, [1, 1],
                                                     ids=[0, 2]))
