"""fp16: a token that outweighs every other one by far, with a value of zero, and a long flat tail, whose small weights
then are the whole result (GPU)."""
import numpy as np
import pytest
import torch

from paged_reference import attention
from slotstream_b200.kernels.paged_attention import attn_decode, attn_prefill, workspace_bytes

pytestmark = pytest.mark.gpu
# Small weights are rounded by up to this part of the largest one: fp16 is exact to 2^-25 near zero, and the largest weight is
# at 2^15, or 2^7 where the maximum may grow by 2^8 before the weights are rescaled.
LEAST_ROWS, LEAST_PROMPT = 2.0 ** -40, 2.0 ** -32


def _case(n, gap, dim, heads, rows, at, room=0, kv=2, ps=16):
    """Every query meets the tokens ``at`` with a score of ``gap``, all others with 0. Values are so large that the result is a
    normal number of the type."""
    pages = -(-n // ps)
    k = torch.zeros(pages, kv, ps, dim, dtype=torch.float16, device="cuda")
    v = 1 + torch.rand(k.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).half() * 0.5
    at = torch.as_tensor(at, device="cuda").reshape(-1)
    v *= 1000 if at.numel() > 1 else 1
    q = torch.ones(rows, heads, dim, dtype=torch.float16, device="cuda")
    k[at // ps, :, at % ps] = gap / dim ** 0.5
    v[at // ps, :, at % ps] = 0
    table = torch.full((1, max(pages, -(-room // ps)) + 1), -1, dtype=torch.int32, device="cuda")
    table[0, :pages] = torch.arange(pages, dtype=torch.int32, device="cuda")
    return q, k, v, table, torch.tensor([n], dtype=torch.int32, device="cuda")


def _where(n, where):
    return {"early": 3, "late": n - 20, "often": torch.arange(3, n, 50)}[where]


def _check(out, lse, q, k, v, table, lens, gap, least):
    o, z, o_tol, z_tol = attention(q, k, v, table, lens, [q.shape[0]])
    # the part of the rounding that is not relative, from all tokens
    o_tol = o_tol + (int(lens[0]) * least * float(v.max()) * torch.exp(gap - z))[..., None]
    assert bool((o > 6.2e-5).all())                          # normal numbers of the type
    err = (out.double() - o).abs()
    assert not bool((err > o_tol).any()), f"off by up to {float((err / o).max()):.3g} of the result"
    assert bool(((lse.double() - z).abs() <= z_tol).all())


# the tokens that stand out: one early, one late, or one in every 50 (so in every tile and every part of a split)
@pytest.mark.parametrize("where", ["early", "late", "often"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,gap", [(30000, 17.6), (30000, 15.0), (3000, 13.0)])
@pytest.mark.parametrize("heads", [4, 24])
def test_decode(dim, n, gap, heads, where):
    """8 and 16 rows an item; contexts of 30,000 tokens are split over the GPU, those of 3,000 go whole."""
    q, k, v, table, lens = _case(n, gap, dim, heads, 1, _where(n, where))
    assert (workspace_bytes(dim, 1, 1, heads, 2, 16, table.shape[1]) > 0) == (n > 8192)
    lse = torch.empty(1, 1, heads, device="cuda")
    out = attn_decode(q[None], k, v, table, lens, lse=lse)
    _check(out[0], lse[0], q, k, v, table, lens, gap, LEAST_ROWS)


# the tokens that stand out: one early, one late, or one in every 50 (so in every tile and every part of a split)
@pytest.mark.parametrize("where", ["early", "late", "often"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,gap", [(30000, 17.6), (30000, 15.0), (3000, 13.0)])
def test_prefill(dim, n, gap, where):
    """A last chunk of 5 tokens on the tensor-core kernel."""
    q, k, v, table, lens = _case(n, gap, dim, 4, 5, _where(n, where), room=70000)
    assert workspace_bytes(dim, 1, 5, 4, 2, 16, table.shape[1], prefill=True) > 0
    lse = torch.empty(5, 4, device="cuda")
    out = attn_prefill(q, k, v, table, lens, torch.tensor([0, 5], dtype=torch.int32, device="cuda"), lse=lse)
    _check(out, lse, q, k, v, table, lens, gap, LEAST_PROMPT)


@pytest.mark.parametrize("heads", [2, 8])
@pytest.mark.parametrize("rise", [3.0, 30.0, 300.0])
def test_weights_that_grow_along_the_cache(heads, rise):
    """Scores that rise from tile to tile by less, and by more, than the step at which the maximum is moved: no weight
    overflows the type."""
    n, dim = 4096, 128
    q, k, v, table, lens = _case(n, 0.0, dim, heads, 40, 3, room=70000)
    k.copy_(torch.linspace(0, rise, n, device="cuda").view(-1, 1, 16, 1) / dim ** 0.5)
    v.copy_(torch.randn(v.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(2)))
    starts = torch.from_numpy(np.array([0, 40], np.int32)).cuda()
    lse = torch.empty(40, heads, device="cuda")
    out = attn_prefill(q, k, v, table, lens, starts, lse=lse)
    o, z, o_tol, z_tol = attention(q, k, v, table, lens, [40])
    assert bool(((out.double() - o).abs() <= o_tol).all()) and bool(((lse.double() - z).abs() <= z_tol).all())
    out = attn_decode(q[-1:][None], k, v, table, lens)
    assert bool(((out[0].double() - o[-1:]).abs() <= o_tol[-1:]).all())
