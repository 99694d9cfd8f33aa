"""The paged K/V cache on the GPU: calls at the corners of what its interface allows."""

import pytest
import torch

from test_paged_cache_gpu import BF16, F16, F32, check, filled, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("length", [10, 300])                         # (items whole and cut)
@pytest.mark.parametrize("few_first", [True, False])
@pytest.mark.parametrize("dtype, tokens, rows, kv_heads", [(BF16, 20, 40, 8), (F16, 9, 80, 8), (F32, 20, 40, 8), (BF16, 48, 60, 4), (F16, 90, 60, 4)])
def test_neighbouring_rows_of_one_sequence_that_end_apart(dtype, tokens, rows, kv_heads, few_first, length):
    """More items than CTAs, so that runs go from one row to the next.  Rows of one token see nothing of the pages behind theirs, whatever those hold."""
    cache, _ = filled([length], [tokens], dtype=dtype, kv_heads=kv_heads, head_dim=64, page_tokens=8 if tokens < 16 else 16)
    q = torch.randn(rows, tokens, kv_heads, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(5)).to(dtype)
    counts = ([1, tokens] if few_first else [tokens, 1]) * (rows // 2)
    clean = check(cache, q, None, counts, [0] * rows)
    behind = cache.table[0, -(-(length + 1) // cache.page_tokens):cache.held[0].item()].long()
    cache.pool[:, :, behind] = float("nan")
    again = cache.attend(0, q, counts=ints(counts), slots=ints([0] * rows))
    few = torch.tensor(counts, device="cuda") == 1
    assert behind.numel() > 0 and torch.equal(clean[few], again[few])
