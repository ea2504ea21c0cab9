"""Attention over the paged cache against its definition in 64 bits (GPU)."""
import numpy as np
import pytest
import torch

from paged_reference import assert_attention, attention
from slotstream_b200.kernels.paged_attention import attn_decode, attn_prefill, workspace_bytes

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _cache(lengths, kv, dim, ps, dtype, seed=0, layers=2, layer=1, spare=3, room=0):
    """Pages dealt at random, the slots past each length filled with NaN; returns strided k / v views and the table, which
    has room for ``room`` tokens a sequence."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    held = [-(-n // ps) for n in lengths]
    pages, mp = sum(held) + spare, max(held + [1, -(-room // ps)]) + 1
    pool = torch.full((pages, layers, 2, kv, ps, dim), float("nan"), dtype=dtype, device="cuda")
    order = np.random.default_rng(seed).permutation(pages)
    table = np.full((len(lengths), mp), -1, np.int32)
    at = 0
    for s, (n, h) in enumerate(zip(lengths, held)):
        table[s, :h] = order[at:at + h]
        at += h
        for j in range(h):
            m = min(ps, n - j * ps)
            pool[int(table[s, j]), layer, :, :, :m] = torch.randn(2, kv, m, dim, device="cuda", generator=g,
                                                                  dtype=torch.float32).to(dtype)
    return (pool[:, layer, 0], pool[:, layer, 1], torch.from_numpy(table).cuda(),
            torch.tensor(lengths, dtype=torch.int32, device="cuda"), g)


def _q(g, rows, heads, kv, dim, dtype):
    """Queries inside a wider projection output: strided, not contiguous."""
    both = torch.randn(rows, heads + 2 * kv, dim, device="cuda", generator=g, dtype=torch.float32).to(dtype)
    return both[:, :heads] * 1 if rows == 0 else both[:, :heads]


def _decode(lengths, q_len, heads, kv, dim, ps, dtype, window=0, sinks=0, seed=0, room=0):
    k, v, table, lens, g = _cache(lengths, kv, dim, ps, dtype, seed, room=room)
    n = len(lengths)
    q = _q(g, n * q_len, heads, kv, dim, dtype)
    lse = torch.full((n, q_len, heads), 7.0, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = attn_decode(q.unflatten(0, (n, q_len)), k, v, table, lens, lse=lse, window=window, sinks=sinks, err=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    assert_attention(out.flatten(0, 1), lse.flatten(0, 1), attention(q, k, v, table, lens, [q_len] * n, window, sinks))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv", [(8, 1), (6, 2), (4, 4), (40, 2)])
def test_decode_one_token(dtype, dim, heads, kv):
    _decode([1, 0, 17, 300, 1025], 1, heads, kv, dim, 16, dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv,q_len", [(8, 2, 1), (24, 2, 1), (3, 1, 5)])
def test_decode_split_over_the_gpu(dtype, dim, heads, kv, q_len):
    """Tables with room for long sequences: the tiles are split evenly over the blocks and joined."""
    assert workspace_bytes(dim, 5, 5 * q_len, heads, kv, 16, 40000 // 16) > 0
    _decode([1, 0, 17, 300, 2049], q_len, heads, kv, dim, 16, dtype, room=40000)


@pytest.mark.parametrize("ps", [1, 5, 8, 24, 100, 128])
@pytest.mark.parametrize("dim", [64, 256])
def test_decode_page_sizes(ps, dim):
    _decode([333, 64, ps, ps + 1, 2 * ps - 1], 1, 8, 2, dim, ps, BF)


@pytest.mark.parametrize("q_len", [1, 2, 3, 5])
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (100, 4), (64, 70), (5000, 4)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_decode_window_and_verify(q_len, window, sinks, dim):
    _decode([0, 1, 2, 130, 700, 1111], q_len, 12, 2, dim, 24, BF, window, sinks)


def test_decode_rows_past_a_tile():
    """64 and 128 query rows per key head: several row blocks."""
    _decode([500, 3], 4, 32, 2, 128, 16, HF)
    _decode([500, 3], 8, 16, 1, 256, 16, BF, 100, 4)


def test_decode_many_sequences_and_a_long_one():
    rng = np.random.default_rng(3)
    _decode([9000] + rng.integers(0, 40, 300).tolist(), 1, 4, 2, 128, 16, BF)
    _decode([20011], 1, 2, 1, 64, 32, HF)


def _prefill(lengths, new, heads, kv, dim, ps, dtype, window=0, sinks=0, seed=0, ids=None, room=0):
    k, v, table, lens, g = _cache(lengths, kv, dim, ps, dtype, seed, room=room)
    rows = sum(new)
    if room or window:      # the tensor-core kernel's workspace, or none: which of the two kernels runs
        big = workspace_bytes(dim, len(new), rows, heads, kv, ps, table.shape[1], window, sinks, prefill=True) > 0
        assert big == (room > 0)
    q = _q(g, rows, heads, kv, dim, dtype)
    starts = torch.from_numpy(np.cumsum([0] + new).astype(np.int32)).cuda()
    lse = torch.full((rows, heads), 7.0, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    idt = None if ids is None else torch.tensor(ids, dtype=torch.int32, device="cuda")
    out = attn_prefill(q, k, v, table, lens, starts, lse=lse, window=window, sinks=sinks, err=err, ids=idt)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    assert_attention(out, lse, attention(q, k, v, table, lens, new, window, sinks, ids=ids))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv", [(2, 2), (6, 2), (8, 1), (5, 1)])
def test_prefill_ragged(dtype, dim, heads, kv):
    _prefill([1, 37, 130, 257, 5], [1, 37, 129, 100, 0], heads, kv, dim, 16, dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv", [(2, 2), (6, 2), (8, 1), (5, 1), (32, 1)])
@pytest.mark.parametrize("ps", [16, 24])
def test_prefill_ragged_on_tcgen05(dtype, dim, heads, kv, ps):
    """Tables with room for long prompts go to the tcgen05 kernel: pages in boxes (16) and row by row (24), groups that
    divide its 128 rows and others."""
    _prefill([1, 37, 130, 257, 5, 700], [1, 37, 129, 100, 0, 3], heads, kv, dim, ps, dtype, room=20000)


@pytest.mark.parametrize("ps", [8, 32, 64, 128, 512])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prefill_boxes_of_every_page_size(ps, dim):
    _prefill([600, 131], [300, 131], 4, 1, dim, ps, BF, room=20000)


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (100, 0), (128, 300), (4000, 1)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prefill_window(window, sinks, dim):
    _prefill([300, 110], [113, 110], 4, 2, dim, 24, BF, window, sinks)


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (100, 0), (128, 300)])
@pytest.mark.parametrize("dim,ps", [(64, 16), (128, 32), (256, 16), (128, 12)])
def test_prefill_window_on_tcgen05(window, sinks, dim, ps):
    _prefill([1500, 700], [900, 700], 16, 4, dim, ps, BF, window, sinks, room=1)


@pytest.mark.parametrize("ps", [1, 7, 64, 200])
def test_prefill_page_sizes_and_ids(ps):
    _prefill([300, 50, 411], [40, 411], 4, 1, 128, ps, BF, ids=[1, 2])
    _prefill([300, 50, 411], [40, 411], 4, 1, 128, ps, BF, ids=[1, 2], room=20000)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("falling", [False, True])
def test_scores_that_rise_or_fall_along_the_cache(dim, falling):
    """Keys growing (or shrinking) with the position: the running maximum rises by far more than one step, over and over
    (or not at all after the first tile), in some rows and not in others."""
    n, new, heads, kv = 1500, 200, 4, 2
    k, v, table, lens, g = _cache([n], kv, dim, 16, BF)
    ramp = torch.linspace(0, 12, n, device="cuda")
    ramp = ramp.flip(0) if falling else ramp
    for t in range(0, n, 16):
        m = min(16, n - t)
        k[int(table[0, t // 16]), :, :m] *= ramp[t:t + m, None].to(BF)
    q = _q(g, new, heads, kv, dim, BF)
    q[::3] *= 0.01
    starts = torch.tensor([0, new], dtype=torch.int32, device="cuda")
    lse, ref = torch.empty(new, heads, device="cuda"), attention(q, k, v, table, lens, [new])
    wide = torch.cat([table, torch.full((1, 1500), -1, dtype=torch.int32, device="cuda")], 1)   # room for 25,000 tokens
    for t in (table, wide):                                                                     # both kernels
        out = attn_prefill(q, k, v, t, lens, starts, lse=lse)
        assert_attention(out, lse, ref)
        out = attn_decode(q[-3:][None], k, v, t, lens, lse=lse[None, -3:])
        assert_attention(out[0], lse[-3:], [x[-3:] for x in ref])


def test_prefill_long_context_few_rows():
    _prefill([9001], [3], 4, 2, 128, 32, BF)
    _prefill([6000], [17], 16, 2, 256, 16, HF, 5000, 8, room=1)


@pytest.mark.parametrize("room", [0, 20000])
def test_prefill_more_queries_than_tokens_sees_nothing(room):
    _prefill([3, 0], [8, 4], 4, 2, 64, 16, BF, room=room)


@pytest.mark.parametrize("room", [0, 20000])
def test_prefill_missing_page_reads_as_zeros_and_is_reported(room):
    k, v, table, lens, g = _cache([700], 1, 128, 16, BF, room=room)
    q = _q(g, 200, 4, 1, 128, BF)
    starts = torch.tensor([0, 200], dtype=torch.int32, device="cuda")
    bad = table.clone()
    bad[0, 5], bad[0, 40] = -1, 10 ** 6
    err, lse = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.empty(200, 4, device="cuda")
    out = attn_prefill(q, k, v, bad, lens, starts, lse=lse, err=err)
    assert int(err.item()) == 128
    none = torch.zeros_like(k[:1])
    bad[0, 5] = bad[0, 40] = k.shape[0]
    assert_attention(out, lse, attention(q, torch.cat([k, none]), torch.cat([v, none]), bad, lens, [200]))


def test_ids_choose_table_rows_and_bad_ids_read_as_empty():
    k, v, table, lens, g = _cache([40, 90, 17], 2, 64, 16, BF)
    q = _q(g, 3, 4, 2, 64, BF).unflatten(0, (3, 1))
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    ids = torch.tensor([2, 5, 0], dtype=torch.int32, device="cuda")
    out = attn_decode(q, k, v, table, lens, ids=ids, err=err)
    ref = attn_decode(q[[0, 2]].contiguous(), k, v, table[[2, 0]].contiguous(), lens[[2, 0]].contiguous())
    assert torch.equal(out[[0, 2]], ref) and bool((out[1] == 0).all())
    assert int(err.item()) == 64


def test_missing_page_reads_as_zeros_and_is_reported():
    k, v, table, lens, g = _cache([70], 1, 64, 16, BF)
    q = _q(g, 1, 4, 1, 64, BF).unflatten(0, (1, 1))
    bad = table.clone()
    bad[0, 1] = 10 ** 6
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = attn_decode(q, k, v, bad, lens, err=err)
    assert int(err.item()) == 128
    pool = torch.zeros_like(k[:1])
    k2, v2 = torch.cat([k, pool]), torch.cat([v, pool])
    bad[0, 1] = k2.shape[0] - 1
    ref = attention(q[0], k2, v2, bad, lens, [1])
    assert bool(((out[0].double() - ref[0]).abs() <= ref[2]).all())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("room", [0, 20000])
def test_other_orders_of_the_cache_and_of_the_queries(dim, room):
    """Token-major pages [pages, page, heads, dim], pages apart by more than their size, and head-major queries."""
    k, v, table, lens, g = _cache([300, 77], 2, dim, 16, BF, room=room)
    q = _q(g, 250, 8, 2, dim, BF)
    starts = torch.tensor([0, 200, 250], dtype=torch.int32, device="cuda")
    lse = torch.empty(250, 8, device="cuda")
    ref = attention(q, k, v, table, lens, [200, 50])
    wide = torch.zeros(k.shape[0], 3, 16, 2, dim, dtype=BF, device="cuda")
    wide[:, 0], wide[:, 2] = k.transpose(1, 2), v.transpose(1, 2)
    k2, v2 = wide[:, 0].transpose(1, 2), wide[:, 2].transpose(1, 2)
    q2 = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert not k2.is_contiguous() and not q2.is_contiguous()
    for kk, vv, qq in ((k2, v2, q), (k, v, q2), (k2, v2, q2)):
        out = attn_prefill(qq, kk, vv, table, lens, starts, lse=lse)
        assert out.is_contiguous()
        assert_attention(out, lse, ref)
        out = attn_decode(qq[[199, 249]][:, None].contiguous() if qq is q else qq[[199, 249]][:, None], kk, vv, table, lens)
        o, _, tol, _ = ref
        assert bool(((out[:, 0].double() - o[[199, 249]]).abs() <= tol[[199, 249]]).all())


def test_pages_behind_the_window_are_not_read():
    """The pages between the sinks and the window may be gone (-1): no error, the same result."""
    k, v, table, lens, g = _cache([700], 2, 128, 16, BF)
    q = _q(g, 1, 4, 2, 128, BF).unflatten(0, (1, 1))
    full = attn_decode(q, k, v, table, lens, window=100, sinks=4)
    gone = table.clone()
    gone[0, 1:(700 - 100) // 16] = -1
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert torch.equal(attn_decode(q, k, v, gone, lens, window=100, sinks=4, err=err), full)
    assert int(err.item()) == 0


def test_results_repeat_and_a_batch_equals_itself_in_a_graph():
    k, v, table, lens, g = _cache([700, 30, 9000], 2, 128, 16, BF)
    q = _q(g, 3, 16, 2, 128, BF).unflatten(0, (3, 1))
    assert table.shape[1] * 16 > 8 * 8 * 128          # a table that calls for the split over blocks, with its workspace
    ws = torch.empty(workspace_bytes(128, 3, 3, 16, 2, 16, table.shape[1]), dtype=torch.uint8, device="cuda")
    assert ws.numel() > 0
    out, ref = torch.empty(q.shape, dtype=BF, device="cuda"), attn_decode(q, k, v, table, lens)
    graph = torch.cuda.CUDAGraph()
    attn_decode(q, k, v, table, lens, out, ws=ws)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        attn_decode(q, k, v, table, lens, out, ws=ws)
    for _ in range(3):
        out.zero_()
        ws.fill_(255)                       # what an earlier call left in the workspace does not matter
        graph.replay()
        assert torch.equal(out, ref)


def test_on_a_side_stream():
    k, v, table, lens, g = _cache([700, 30], 2, 64, 16, HF)
    q = _q(g, 2, 4, 2, 64, HF).unflatten(0, (2, 1))
    ref = attn_decode(q, k, v, table, lens)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out = attn_decode(q, k, v, table, lens)
    side.synchronize()
    assert torch.equal(out, ref)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 elements, the sequence at its end."""
    ps, kv, dim = 16, 8, 128
    pages = 2 ** 32 // (2 * ps * kv * dim) + 5
    pool = torch.empty(pages, 1, 2, kv, ps, dim, dtype=BF, device="cuda")
    pool[-3:] = torch.randn(3, 1, 2, kv, ps, dim, device="cuda").to(BF)
    table = torch.tensor([[pages - 1, pages - 3, pages - 2]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([43], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 1, 16, dim, device="cuda").to(BF)
    lse = torch.empty(1, 1, 16, device="cuda")
    for out in (attn_decode(q, pool[:, 0, 0], pool[:, 0, 1], table, lens, lse=lse),
                attn_prefill(q[0], pool[:, 0, 0], pool[:, 0, 1], table, lens,
                             torch.tensor([0, 1], dtype=torch.int32, device="cuda"), lse=lse[0])[None]):
        assert_attention(out[0], lse[0], attention(q[0], pool[:, 0, 0], pool[:, 0, 1], table, lens, [1]))
    del pool
    torch.cuda.empty_cache()
