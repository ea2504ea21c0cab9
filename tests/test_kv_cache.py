"""Host side of the paged cache and its attention: refusals that need no GPU, at the Python and the C entries (CPU)."""
import ctypes

import pytest
import torch

from slotstream_b200 import _lib
from slotstream_b200.kernels.paged_attention import attn_decode, attn_prefill
from slotstream_b200.kv_cache import PagedKvCache, state_ints


def _args(dim=64, dtype=torch.bfloat16, kv=2, n=1):
    pages = torch.zeros(4, kv, 16, dim, dtype=dtype)
    return (torch.zeros(n, 1, 4, dim, dtype=dtype), pages, pages.clone(), torch.zeros(n, 2, dtype=torch.int32),
            torch.zeros(n, dtype=torch.int32))


def test_state_size():
    assert state_ints(33, 2, 5) == 2 + 33 + 2 + 10 + 1


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(1, 4, 64, dtype=torch.bfloat16)), "q must be"),
    (dict(q=torch.zeros(1, 1, 4, 64)), "bf16"),
    (dict(q=torch.zeros(1, 1, 4, 128, dtype=torch.bfloat16)[..., ::2]), "contiguous"),
    (dict(k=torch.zeros(4, 2, 16, 64, dtype=torch.float16)), "bf16"),
    (dict(k=torch.zeros(4, 2, 8, 64, dtype=torch.bfloat16)), "must both be"),
    (dict(v=torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16).transpose(1, 2)), "strides"),
    (dict(q=torch.zeros(1, 1, 3, 64, dtype=torch.bfloat16)), "no multiple"),
    (dict(table=torch.zeros(1, 2, dtype=torch.int64)), "page_table"),
    (dict(lengths=torch.zeros(2, dtype=torch.int32)), "lengths"),
    (dict(kw=dict(window=-1)), "negative"),
    (dict(kw=dict(sinks=-1)), "negative"),
    (dict(kw=dict(scale=0.0)), "scale"),
    (dict(kw=dict(scale=float("nan"))), "scale"),
    (dict(kw=dict(ids=torch.zeros(2, dtype=torch.int32))), "ids"),
    (dict(kw=dict(lse=torch.zeros(1, 1, 4, 1))), "lse"),
    (dict(kw=dict(out=torch.zeros(1, 1, 4, 32, dtype=torch.bfloat16))), "out"),
    (dict(kw=dict(err=torch.zeros(2, dtype=torch.int32))), "err"),
])
def test_attention_argument_errors(change, match):
    a = dict(zip(("q", "k", "v", "table", "lengths"), _args()))
    kw = change.pop("kw", {})
    a.update(change)
    with pytest.raises(ValueError, match=match):
        attn_decode(a["q"], a["k"], a["v"], a["table"], a["lengths"], **kw)


def test_prefill_argument_errors():
    q, k, v, table, lens = _args()
    starts = torch.tensor([0, 1], dtype=torch.int32)
    with pytest.raises(ValueError, match="q must be"):
        attn_prefill(q, k, v, table, lens, starts)
    with pytest.raises(ValueError, match="starts"):
        attn_prefill(q[0], k, v, table, lens, starts.long())
    with pytest.raises(ValueError, match="sequences"):
        attn_prefill(q[0], k, v, table, lens, torch.tensor([0, 1, 1], dtype=torch.int32))


@pytest.mark.parametrize("shape,state,seqs", [
    ((4, 1, 2, 2, 16), 30, 2), ((4, 1, 3, 2, 16, 64), 30, 2), ((4, 1, 2, 2, 16, 4), 30, 2),
    ((4, 1, 2, 2, 16, 64), 7, 2), ((4, 1, 2, 2, 16, 64), state_ints(4, 2, 3) + 1, 2)])
def test_cache_argument_errors(shape, state, seqs):
    with pytest.raises(ValueError):
        PagedKvCache.over(torch.zeros(shape, dtype=torch.bfloat16), torch.zeros(state, dtype=torch.int32), seqs)


def test_cache_lives_on_the_gpu():
    with pytest.raises(ValueError, match="CUDA"):
        PagedKvCache.over(torch.zeros(4, 1, 2, 2, 16, 64, dtype=torch.bfloat16),
                          torch.zeros(state_ints(4, 2, 3), dtype=torch.int32), 2)
    with pytest.raises(ValueError, match="at least 1"):
        PagedKvCache(0, 1, 1, 16, 64, 1, 1)


def _rows(**change):
    f = dict(k=64, v=64, k_row=64, k_head=64, v_row=64, v_head=64, rows=1, starts=64, ids=0, kl=64, vl=64, sp=64, sh=64, st=64,
             n=1, kv=1, dim=64)
    f.update(change)
    return _lib.KV_ROWS.pack(*f.values())


def _c_cache(**change):
    f = dict(pool=4096, page_bytes=4096, pages=4, page_size=16, seqs=2, max_pages=3, lengths=64, refs=64, free_words=64,
             table=64, err=64, scratch=64)
    f.update(change)
    return _lib.KvCacheStruct(**f)


@pytest.mark.parametrize("change", [
    dict(pool=None), dict(pool=4104), dict(page_bytes=8), dict(page_bytes=0), dict(pages=0), dict(pages=(1 << 20) + 1),
    dict(page_size=0), dict(seqs=0), dict(seqs=65537), dict(max_pages=0), dict(max_pages=1 << 30), dict(lengths=None),
    dict(refs=None), dict(free_words=None), dict(table=None), dict(scratch=None)])
def test_c_entry_refuses_a_bad_cache(change):
    """Checked on the host before any launch: every call gives SSB_EINVAL."""
    c, L = _c_cache(**change), _lib.lib()
    p = ctypes.addressof(c)
    assert L.ssb_kv_extend(p, 64, 64, 1, None) == _lib.SSB_EINVAL
    assert L.ssb_kv_fork(p, 64, 64, 1, None) == _lib.SSB_EINVAL
    assert L.ssb_kv_free(p, 64, None, None, 1, None) == _lib.SSB_EINVAL
    assert L.ssb_kv_compact(p, None) == _lib.SSB_EINVAL
    assert L.ssb_kv_write(p, _rows(), None) == _lib.SSB_EINVAL


def test_c_entry_counts_and_nulls():
    c, L = _c_cache(), _lib.lib()
    p = ctypes.addressof(c)
    assert L.ssb_kv_extend(None, 64, 64, 1, None) == _lib.SSB_EINVAL
    assert L.ssb_kv_extend(p, 64, 64, 0, None) == _lib.SSB_OK
    assert L.ssb_kv_extend(p, 64, 64, 3, None) == _lib.SSB_EINVAL
    assert L.ssb_kv_extend(p, None, 64, 1, None) == _lib.SSB_EINVAL
    assert L.ssb_kv_fork(p, 64, None, 1, None) == _lib.SSB_EINVAL
    assert L.ssb_kv_free(p, 64, 64, None, 1, None) == _lib.SSB_EINVAL
    assert L.ssb_kv_write(p, None, None) == _lib.SSB_EINVAL
    assert L.ssb_kv_write(p, _rows(dim=60), None) == _lib.SSB_EUNSUPPORTED
    assert L.ssb_kv_write(p, _rows(k_row=60), None) == _lib.SSB_EINVAL
    assert L.ssb_kv_write(p, _rows(k=72), None) == _lib.SSB_EINVAL
    assert L.ssb_kv_write(p, _rows(starts=0), None) == _lib.SSB_EINVAL
    assert L.ssb_kv_write(p, _rows(rows=-1), None) == _lib.SSB_EINVAL
    assert L.ssb_kv_write(p, _rows(rows=0), None) == _lib.SSB_OK
    assert L.ssb_kv_scratch_ints(0, 1) == _lib.SSB_EINVAL


def _attn_args(**change):
    f = dict(q=64, k=64, v=64, qs=64, qt=64, qh=64, sp=64, sh=64, st=64, table=64, lengths=64, ids=0, starts=64, out=64, lse=0,
             err=0, ws=64, ws_bytes=0, total=1, q_type=_lib.BF16, n=1, q_len=1, heads=4, kv=2, dim=64, ps=16, pages=4, rows=1,
             mp=3, window=0, sinks=0, scale=1.0)
    f.update(change)
    return _lib.ATTN_ARGS.pack(*f.values())


def test_packed_arguments_have_the_c_layout():
    """The fields' order and alignment, and the sizes of the C structs without their padding at the end."""
    assert _lib.ATTN_ARGS.size == 8 * 19 + 13 * 4 and _lib.KV_ROWS.size == 8 * 14 + 3 * 4


@pytest.mark.parametrize("change,want", [
    (dict(mp=1 << 16), _lib.SSB_EINVAL),                           # no workspace
    (dict(q_type=_lib.F32), _lib.SSB_EINVAL), (dict(dim=96), _lib.SSB_EUNSUPPORTED),
    (dict(q_len=65), _lib.SSB_EUNSUPPORTED), (dict(heads=5), _lib.SSB_EINVAL), (dict(kv=0), _lib.SSB_EINVAL),
    (dict(ps=0), _lib.SSB_EINVAL), (dict(pages=0), _lib.SSB_EINVAL), (dict(rows=0), _lib.SSB_EINVAL),
    (dict(mp=1 << 28), _lib.SSB_EINVAL), (dict(window=-1), _lib.SSB_EINVAL), (dict(sinks=-1), _lib.SSB_EINVAL),
    (dict(st=63), _lib.SSB_EINVAL), (dict(qh=4), _lib.SSB_EINVAL), (dict(k=72), _lib.SSB_EINVAL),
    (dict(scale=-1.0), _lib.SSB_EINVAL), (dict(n=-1), _lib.SSB_EINVAL), (dict(n=0), _lib.SSB_OK), (dict(q_len=0), _lib.SSB_OK),
    (dict(q=0, ws_bytes=1 << 40), _lib.SSB_EINVAL), (dict(ws=0, ws_bytes=1 << 40, mp=1 << 16), _lib.SSB_EINVAL)])
def test_c_attention_refusals(change, want):
    assert _lib.lib().ssb_attn_decode(_attn_args(**change), None) == want


@pytest.mark.parametrize("change,want", [
    (dict(mp=1 << 16), _lib.SSB_EINVAL), (dict(total=-1), _lib.SSB_EINVAL), (dict(total=1 << 30), _lib.SSB_EINVAL),
    (dict(starts=0), _lib.SSB_EINVAL), (dict(dim=32), _lib.SSB_EUNSUPPORTED), (dict(qt=4), _lib.SSB_EINVAL),
    (dict(total=0), _lib.SSB_OK), (dict(n=0), _lib.SSB_OK)])
def test_c_prefill_refusals(change, want):
    assert _lib.lib().ssb_attn_prefill(_attn_args(**change), None) == want


def test_c_null_arguments():
    L, b = _lib.lib(), ctypes.c_int64()
    assert L.ssb_attn_decode(None, None) == L.ssb_attn_prefill(None, None) == _lib.SSB_EINVAL
    assert L.ssb_attn_workspace(None, 0, ctypes.byref(b)) == L.ssb_attn_workspace(_attn_args(), 0, None) == _lib.SSB_EINVAL
    assert L.ssb_attn_workspace(_attn_args(mp=1 << 16), 0, ctypes.byref(b)) == _lib.SSB_OK and b.value > 0
    assert L.ssb_attn_workspace(_attn_args(), 0, ctypes.byref(b)) == _lib.SSB_OK and b.value == 0
