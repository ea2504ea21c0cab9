"""Windows wider than any sequence, up to the largest that is taken, with queries before the sequence's start (GPU)."""
import numpy as np
import pytest
import torch

from paged_reference import assert_attention, attention
from slotstream_b200.kernels.paged_attention import attn_decode, attn_prefill
from test_gpu_paged_attention import _cache, _q

pytestmark = pytest.mark.gpu
LENGTHS = [1, 2, 3, 0, 40, 700]


@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 0), (2 ** 31 - 1, 5), (2 ** 31 - 2, 0), (2 ** 31 - 4, 1)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("room", [0, 40000])
def test_decode(window, sinks, dim, room):
    """Both paths of the kernel: items whole, and split over the GPU (tables with room for long sequences)."""
    k, v, table, lens, g = _cache(LENGTHS, 2, dim, 16, torch.bfloat16, room=room)
    n = len(LENGTHS)
    for q_len in (4, 7):
        q = _q(g, n * q_len, 8, 2, dim, torch.bfloat16)
        lse = torch.full((n * q_len, 8), 7.0, device="cuda")
        out = attn_decode(q.unflatten(0, (n, q_len)), k, v, table, lens, lse=lse.unflatten(0, (n, q_len)), window=window,
                          sinks=sinks)
        assert_attention(out.flatten(0, 1), lse, attention(q, k, v, table, lens, [q_len] * n, window, sinks))


@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 0), (2 ** 31 - 1, 5), (2 ** 31 - 4, 1)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("room", [0, 20000])
def test_prefill(window, sinks, dim, room):
    k, v, table, lens, g = _cache(LENGTHS, 2, dim, 16, torch.bfloat16, room=room)
    new = [9, 4, 70, 5, 44, 30]
    q = _q(g, sum(new), 8, 2, dim, torch.bfloat16)
    lse = torch.full((sum(new), 8), 7.0, device="cuda")
    starts = torch.from_numpy(np.cumsum([0] + new).astype(np.int32)).cuda()
    out = attn_prefill(q, k, v, table, lens, starts, lse=lse, window=window, sinks=sinks)
    assert_attention(out, lse, attention(q, k, v, table, lens, new, window, sinks))
