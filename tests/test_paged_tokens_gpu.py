"""PagedDecoder: counts that its tokens do not reach, and prompts that the cache cannot hold."""

from __future__ import annotations

import numpy as np
import pytest

from tests.conftest import gpu_available
from tests.gpu_util import announce
from tests.test_paged_decoder_gpu import make

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]


def _prompts(seed, *lengths):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, 512, n).tolist() for n in lengths]


def test_a_count_past_the_tokens_refuses_its_request():
    """Counts on the GPU, eagerly and in a captured step: nothing of the request is written and its length stays;
    the others' logits are those of a step in which it has no new tokens."""
    import torch

    from ironmule_amd.paged import PagedCache, PagedDecoder
    announce("paged counts past the tokens")
    weights = make("decoder", 21)
    models = [PagedDecoder(weights, PagedCache(weights.config, 3, 64, 16, 60, "cuda", page_size=16)) for _ in range(3)]
    for m in models:
        m.prefill(_prompts(1, 9, 20, 3))
    tokens = torch.tensor([[5, 6], [7, 8], [9, 10]], dtype=torch.int32, device="cuda")
    counts = torch.tensor([2, 3, 1], dtype=torch.int32, device="cuda")
    kept = models[0].cache.tables.clone()
    got = models[0].extend(tokens, counts, rows=6)
    want = models[1].extend(tokens, [2, 0, 1], rows=6)
    assert models[0].cache.status.tolist() == [0, 2, 0] and models[0].cache.lengths.tolist() == [11, 20, 4]
    assert torch.isnan(got[1]).all() and torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    assert torch.equal(models[0].cache.tables[1], kept[1])
    got = models[0].extend([[5], [], [9, 10]], torch.tensor([2, 1, 2], device="cuda"))  # lists, each with its own length
    assert models[0].cache.status.tolist() == [2, 2, 0] and models[0].cache.lengths.tolist() == [11, 20, 6]
    assert torch.isnan(got[:2]).all() and got[2].isfinite().all()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = models[2].extend(tokens, counts, rows=6)
    for step in range(3):  # the second time every count fits, the third the first one does not
        counts.copy_(torch.tensor([[2, 3, 1], [2, 2, 2], [2**31 - 1, 1, 1]][step], dtype=torch.int32))
        graph.replay()
        if step:
            eager = models[1].extend(tokens, [[2, 2, 2], [0, 1, 1]][step - 1], rows=6)
            assert torch.equal(out.nan_to_num(9.0), eager.nan_to_num(9.0))
        torch.cuda.synchronize()
        assert models[2].cache.lengths.tolist() == models[1].cache.lengths.tolist()
        assert models[2].cache.status.tolist() == [[0, 2, 0], [0, 0, 0], [2, 0, 0]][step]


def test_a_refused_prompt_leaves_what_it_begins_with():
    """A chunk that does not fit ends its request's prompt, though the last and smaller one would fit; the other
    prompts go on, and the rest can be taken later where pages have become free."""
    import torch

    from ironmule_amd.paged import PagedCache, PagedDecoder
    announce("paged prompts that do not fit")
    weights = make("decoder", 22)
    cache = PagedCache(weights.config, 3, 192, 10, 64, "cuda", page_size=16)
    model = PagedDecoder(weights, cache)
    roomy = PagedDecoder(weights, PagedCache(weights.config, 3, 192, 40, 64, "cuda", page_size=16))
    held, long, other = _prompts(2, 64, 150, 5)
    model.prefill([held, [], []])  # 4 of the 10 pages; 64 tokens of `long` take 4, 2 are left
    with pytest.raises(RuntimeError):
        model.prefill([[], long, other])
    assert cache.lengths.tolist() == [64, 64, 5]
    cache.release([0, 2])  # 6 pages, as many as the rest takes
    got = model.prefill([[], long[64:], []])
    assert cache.lengths.tolist() == [0, 150, 0]
    roomy.prefill([held, [], []])
    roomy.prefill([[], long[:64], []])
    roomy.cache.release([0])
    want = roomy.prefill([[], long[64:], []])
    assert torch.equal(got[1], want[1])
