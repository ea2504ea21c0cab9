"""Paths of the attention kernels that need particular sizes: the split with windows, many sequences in one launch, cut items
when piece slots run out; repeatability and capture of prompts (GPU)."""
import numpy as np
import pytest
import torch

from paged_reference import assert_attention, attention
from slotstream_b200.kernels.paged_attention import attn_decode, attn_prefill, workspace_bytes
from test_gpu_paged_attention import _cache, _q

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv,q_len", [(8, 2, 1), (8, 2, 2), (12, 2, 3)])
@pytest.mark.parametrize("window,sinks", [(9000, 0), (9000, 300), (8200, 4)])
def test_split_decode_with_window(dtype, dim, heads, kv, q_len, window, sinks):
    """Windows of more tiles than go whole: sink tiles and window tiles divided over the blocks, sequences longer and shorter
    than the window, one with fewer tokens than queries."""
    lengths = [20000, 9100, 5000, 9001, 2, 0]
    n = len(lengths)
    k, v, table, lens, g = _cache(lengths, kv, dim, 16, dtype)
    assert workspace_bytes(dim, n, n * q_len, heads, kv, 16, table.shape[1], window, sinks) > 0
    q = _q(g, n * q_len, heads, kv, dim, dtype)
    lse = torch.full((n, q_len, heads), 7.0, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = attn_decode(q.unflatten(0, (n, q_len)), k, v, table, lens, lse=lse, window=window, sinks=sinks, err=err)
    assert int(err.item()) == 0
    assert_attention(out.flatten(0, 1), lse.flatten(0, 1), attention(q, k, v, table, lens, [q_len] * n, window, sinks))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_sequences_in_one_launch(dim):
    """More sequences than a block has threads, each item whole."""
    lengths = np.random.default_rng(5).integers(0, 300, 290).tolist()
    k, v, table, lens, g = _cache(lengths, 2, dim, 16, BF)
    assert workspace_bytes(dim, 290, 290, 8, 2, 16, table.shape[1]) == 0
    q = _q(g, 290, 8, 2, dim, BF)
    lse = torch.full((290, 8), 7.0, device="cuda")
    out = attn_decode(q[:, None], k, v, table, lens, lse=lse[:, None])
    assert_attention(out[:, 0], lse, attention(q, k, v, table, lens, [1] * 290))


@pytest.mark.parametrize("dim,heads,kv", [(256, 32, 4), (128, 32, 8)])
def test_more_pieces_wanted_than_there_are_slots(dim, heads, kv):
    """512 tokens after 6,000: a few items at the end of the list stay whole. Rows of every part of the chunk."""
    new, n = 512, 6512
    k, v, table, lens, g = _cache([n], kv, dim, 16, BF, layers=1, layer=0)
    q = _q(g, new, heads, kv, dim, BF)
    lse = torch.full((new, heads), 7.0, device="cuda")
    starts = torch.tensor([0, new], dtype=torch.int32, device="cuda")
    out = attn_prefill(q, k, v, table, lens, starts, lse=lse)
    rows = list(range(0, new, 37)) + [1, 31, 32, 63, 64, 127, 128, 255, 256, new - 1]
    ref = attention(q[rows], k, v, table.expand(len(rows), -1),
                    torch.tensor([n - new + r + 1 for r in rows], dtype=torch.int32), [1] * len(rows))
    assert_attention(out[rows], lse[rows], ref)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("ps", [16, 24])
def test_prompts_repeat_bit_for_bit(dim, ps):
    """Units are taken by whichever block is free; cut items are joined in their own order."""
    k, v, table, lens, g = _cache([6000, 700, 1, 3000], 2, dim, ps, BF)
    q = _q(g, 700, 8, 2, dim, BF)
    starts = torch.tensor([0, 300, 400, 401, 700], dtype=torch.int32, device="cuda")
    assert workspace_bytes(dim, 4, 700, 8, 2, ps, table.shape[1], prefill=True) > 0
    lse = torch.empty(700, 8, device="cuda")
    out = attn_prefill(q, k, v, table, lens, starts, lse=lse)
    for _ in range(10):
        again = torch.empty_like(lse)
        assert torch.equal(attn_prefill(q, k, v, table, lens, starts, lse=again), out) and torch.equal(again, lse)


@pytest.mark.parametrize("room", [0, 20000])
@pytest.mark.parametrize("ps", [16, 24])
def test_prompts_can_be_captured(room, ps):
    """Both kernels, with the caller's workspace; later replays see the lengths, tables and queries of their time."""
    k, v, table, lens, g = _cache([300, 130], 2, 128, ps, BF, room=room)
    q = _q(g, 140, 8, 2, 128, BF)
    starts = torch.tensor([0, 100, 140], dtype=torch.int32, device="cuda")
    need = workspace_bytes(128, 2, 140, 8, 2, ps, table.shape[1], prefill=True)
    assert (need > 0) == (room > 0)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
    out, lse = torch.empty(140, 8, 128, dtype=BF, device="cuda"), torch.empty(140, 8, device="cuda")
    attn_prefill(q, k, v, table, lens, starts, out, lse=lse, ws=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attn_prefill(q, k, v, table, lens, starts, out, lse=lse, ws=ws)
    for step in range(3):
        if step:
            lens -= 7
            starts[1] += 9
            q.copy_(torch.randn(q.shape, device="cuda", generator=g))
        out.zero_()
        if ws is not None:
            ws.fill_(255)
        graph.replay()
        new = [100 + 9 * step, 40 - 9 * step]
        assert_attention(out, lse, attention(q, k, v, table, lens, new))
