"""Appends to a paged cache that are refused before their device is looked at (no GPU)."""

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
