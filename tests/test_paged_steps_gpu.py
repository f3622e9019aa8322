"""Steps of a beam search in one captured graph (selection, reordering, the next tokens through the model), and
tokens outside the vocabulary."""

from __future__ import annotations

import numpy as np
import pytest

from tests.conftest import gpu_available
from tests.gpu_util import announce
from tests.test_paged_decoder_gpu import make

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]


@pytest.mark.parametrize("kind", ["decoder", "gemma3"])
def test_a_captured_search_step_gives_the_eager_search(kind):
    """Nine replays, with eager work of the other search and synchronizations between them; pages are shared,
    copied and given back as the beams go."""
    import torch

    from ironmule_amd import _native
    from ironmule_amd.paged import PagedCache, PagedDecoder
    announce("captured search steps", kind)
    weights = make(kind, 31)
    groups, beams, steps, eos = 2, 4, 9, 7
    rng = np.random.default_rng(8)
    prompts = [rng.integers(0, 512, n).tolist() for n in (29, 15)]
    models = [PagedDecoder(weights, PagedCache(weights.config, groups * beams, 128, 60, 64, "cuda", page_size=16))
              for _ in range(2)]
    first = [prompts[r // beams] if r % beams == 0 else [] for r in range(groups * beams)]
    states = []
    for m in models:
        states.append(dict(logits=m.prefill(first).clone(), scores=torch.zeros(groups * beams, device="cuda"),
                           finished=torch.zeros(groups * beams, dtype=torch.int32, device="cuda")))

    def step(m, s):
        scores, parents, tokens, ended = (t.reshape(-1) for t in _native.beam_select(
            s["logits"], s["scores"], beams, beams, finished=s["finished"], eos=eos))
        m.cache.reorder(parents)
        going = ((parents >= 0) & (ended == 0)).int()
        logits = m.extend(tokens.clamp(min=0)[:, None], going, rows=groups * beams)
        for name, value in (("logits", logits), ("scores", scores), ("finished", ended)):
            s[name].copy_(value)
        return parents, tokens

    kept = [t.clone() for t in states[0].values()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        made = step(models[0], states[0])
    assert all(torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0)) for a, b in zip(kept, states[0].values()))
    for i in range(steps):
        graph.replay()
        want = step(models[1], states[1])
        torch.cuda.synchronize()
        for a, b in zip((*made, *states[0].values()), (*want, *states[1].values())):
            assert torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0)), i
        a, b = (m.cache for m in models)
        assert torch.equal(a.tables, b.tables) and torch.equal(a.refs, b.refs) and torch.equal(a.lengths, b.lengths)
        assert not a.status.any()
    held = models[0].cache.tables[models[0].cache.tables >= 0]
    assert torch.equal(torch.bincount(held, minlength=60), models[0].cache.refs.long())


@pytest.mark.parametrize("kind", ["decoder", "gemma3"])
@pytest.mark.parametrize("token", [512, -1, 2**31 - 1, -2**31])
def test_a_token_outside_the_vocabulary_is_its_own_requests_trouble(kind, token):
    """Its request's logits are NaN from then on; the others' are what they are beside a token that exists."""
    import torch

    from ironmule_amd.paged import PagedCache, PagedDecoder
    announce("tokens outside the vocabulary", kind, token)
    weights = make(kind, 32)
    models = [PagedDecoder(weights, PagedCache(weights.config, 3, 128, 30, 64, "cuda", page_size=16)) for _ in range(2)]
    rng = np.random.default_rng(9)
    prompts = [rng.integers(0, 512, n).tolist() for n in (20, 9, 5)]
    outs = []
    for m, bad in zip(models, (token, 3)):
        m.prefill(prompts)
        got = [m.extend([[1], [bad], [2]], [1, 1, 1])]
        got += [m.extend([[4], [5], [6]], [1, 1, 1])]
        got += [m.extend([[7] * 6, [8] * 40, [9]], [6, 40, 1])]
        outs.append(got)
    for a, b in zip(*outs):
        assert torch.isnan(a[1]).all() and b.isfinite().all()
        assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
    models[0].cache.release([1])
    again = models[0].extend([[], prompts[1], []], [0, 9, 0])
    assert again[1].isfinite().all()  # the pages that held NaNs are another request's now
