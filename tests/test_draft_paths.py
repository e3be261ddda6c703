"""Accepted paths that are no indices: a mask would be taken for the indices 0 and 1."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from logkv_amd.streaming import _check_path


@pytest.mark.parametrize("path", [
    torch.tensor([False, True]), [False, True], [[False, True], [False, True]], [True], [0.0, 1.0], torch.tensor([0.0, 1.5]),
    [None], ["0"], torch.zeros(1, 1, 1, dtype=torch.long), np.array([False, True]),
    [torch.tensor(False), torch.tensor(True)], [np.bool_(True)], [[0, 1], 2], [0, [1]]])
def test_no_indices(path):
    with pytest.raises(ValueError, match="path"):
        _check_path(path, 4, 2)


def test_indices_of_other_types():
    assert _check_path(np.array([0, 3]), 4, 2) == [[0, 3]] and _check_path(np.array([[0, 3], [1, 2]]), 4, 2) == [[0, 3], [1, 2]]
    assert _check_path([np.int32(1), torch.tensor(2)], 4, 2) == [[1, 2]]
    rows = _check_path([np.int64(0), torch.tensor(1)], 4, 2)
    assert all(type(i) is int for row in rows for i in row)
    assert _check_path((i for i in (0, 2)), 4, 2) == [[0, 2]]
