"""The counts of a reservation are one for each request: no GPU needed."""

from __future__ import annotations

import pytest
import torch

from ironmule_amd.decode import DecoderConfig
from ironmule_amd.paged import PagedCache


@pytest.mark.parametrize("counts", [[1], 1, [1, 1], [[1, 1, 1]], [], torch.tensor([2], dtype=torch.int32),
                                    torch.tensor(2), torch.ones((3, 1), dtype=torch.int32)])
def test_counts_of_another_shape_are_refused(counts):
    """One number is not taken for every request."""
    cfg = DecoderConfig(hidden=256, layers=1, heads=4, kv_heads=2, head_dim=128, intermediate=512, vocab=512)
    cache = PagedCache(cfg, 3, 64, 8, 16, "cpu", page_size=16)
    with pytest.raises(ValueError, match="counts"):
        cache.reserve(counts)
    assert not cache.counts.any()
