"""Arguments of appends to a paged cache, refused or as they are passed on (no GPU)."""

from __future__ import annotations

import pytest
import torch

from logkv_amd import log_kv_paged_append


def test_no_groups():
    """Queries beside rows of no group would come back as memory that nothing has written."""
    q, k, pages = torch.ones(2, 4, 3, 64), torch.ones(2, 0, 3, 64), torch.ones(8, 0, 16, 64)
    table = torch.zeros(2, 2, dtype=torch.int32)
    for kw in (dict(q=q, frequencies=torch.ones(32)), dict(q=q), {}):
        with pytest.raises(ValueError, match="group"):
            log_kv_paged_append(k, k, pages.bfloat16(), pages.bfloat16(), table, 0, **kw)


def test_counts_beyond_32_bits():
    """int64 lengths and counts are held to what int32 can say, not cut to their lower half."""
    from logkv_amd.paged_attention import _check_counts
    from logkv_amd.row_attention import _lengths

    given = torch.tensor([2 ** 32 + 5, -2 ** 32 + 5, 2 ** 31, 7, -3])
    want = [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 7, -3]
    lengths, address, stride, add = _lengths(given, 5, 100, -1)
    assert lengths.tolist() == want and lengths.dtype == torch.int32 and (address, stride, add) == (lengths.data_ptr(), 1, 0)
    assert _check_counts(given, 5, -1).tolist() == want
    every_other = torch.tensor([[1, 2], [3, 4]], dtype=torch.int32)[:, 1]
    assert _lengths(every_other, 2, 100, -1)[0].tolist() == [2, 4] and _check_counts(every_other, 2, -1).is_contiguous()
