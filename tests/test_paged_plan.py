"""How an attention over pages is planned, by the workspace that it asks for: no GPU needed."""

from __future__ import annotations

import os

import pytest

from ironmule_amd import _native


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_native.LIB_PATH):
        from ironmule_amd import build
        build.build()
    return _native.lib()


@pytest.mark.parametrize("requests", [2, 3])
def test_long_requests_do_not_count_as_tiles_of_few_queries(lib, requests):
    """Beside a chunk the requests of few queries have two tiles each at most, however many rows the chunk has.
    (Up to 1024 keys the chunk's own tiles are whole and ask for nothing, so that what is asked for is theirs.)"""
    needs = {lib.imq_paged_attention_workspace(rows, requests, 4, 1, 128, 1024, 0) for rows in (40, 60, 80, 100)}
    # two tiles of 32 + 2 blocks for each request: parts of 8, two partial results of 16 queries for each part
    parts = -(-2 * requests * 34 // 8)
    assert needs == {2 * parts * 16 * (128 * 4 + 8)}
