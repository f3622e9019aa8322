"""PagedDecoder: prompts in chunks, mixed steps, shared prefixes, beam search and captured steps over a
paged cache, against the decode oracle (float64) and against steps that share nothing.

The bar against the oracle is derived per run: the oracle's own composition with every activation rounded to
bf16 and without any rounding lie `d` apart.  The GPU rounds at the oracle's points (and the
attention's probabilities besides, one rounding among ten a layer); a value that rounds the other way
sets off others, so it lies as far from the exact composition as the rounded oracle does, and within
2 d of that.  With these
weights 2 d is 0.06 and 0.11; an early token that is missing or another moves a logit by 0.35 to 0.96,
a window that is one too wide by 0.89."""

import numpy as np
import pytest

from tests.conftest import gpu_available
from tests.gpu_util import announce, oracle_decoder, oracle_gemma3

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]

CAPACITY = 128


def centred(weights):
    """The weights with every bias at -7.5 scales: products of both signs, so that the logits depend on
    every key (with biases of one sign the common term hides them)."""
    import torch

    def centre(quant):
        w, s, b = quant
        return w, s, (-7.5 * s.float()).to(torch.bfloat16)

    for layer in weights.layers:
        for name in weights.config.projections:
            layer[name] = centre(layer[name])
    weights.embed = centre(weights.embed)
    return weights


def make(kind, seed, device="cuda"):
    from ironmule_amd.decode import DecoderConfig, random_weights
    from ironmule_amd.gemma3 import Gemma3Config, random_gemma3_weights
    if kind == "decoder":
        cfg = DecoderConfig(hidden=256, layers=2, heads=4, kv_heads=2, head_dim=128, intermediate=512, vocab=512)
        return centred(random_weights(cfg, device, seed=seed))
    cfg = Gemma3Config(hidden=512, layers=3, heads=4, kv_heads=2, head_dim=256, intermediate=1024, vocab=512, window=21,
                       pattern=3)
    return centred(random_gemma3_weights(cfg, device, seed=seed))


class Oracle:
    """The logits after every token of some requests, rounded (`ref`) and not."""

    def __init__(self, weights, kind, slots):
        from oracle import decode_oracle as do
        from oracle import oracle as orc
        self.model = (oracle_decoder if kind == "decoder" else oracle_gemma3)(do, orc, weights)
        self.model.layers = list(self.model.layers)
        self.step = do.decode_step if kind == "decoder" else do.gemma3_decode_step
        c = weights.config
        self.pools = [[np.zeros((slots, c.kv_heads, CAPACITY, c.head_dim)) for _ in range(c.layers)] for _ in range(4)]
        self.at = [0] * slots

    def feed(self, slot, tokens):
        for token in tokens:
            args = [token], [slot], [self.at[slot]]
            ref = self.step(self.model, *self.pools[:2], *args, round_bf16=True)[0]
            exact = self.step(self.model, *self.pools[2:], *args, round_bf16=False)[0]
            self.at[slot] += 1
        return ref, np.abs(ref - exact).max()


def check(got, ref, d, what):
    error = np.abs(got.cpu().numpy().astype(np.float64) - ref).max()
    print(f"[observed] {what}: {error:.3e}, rounding {d:.3e}", flush=True)
    assert error <= 2 * d, (what, error, d)


@pytest.mark.parametrize("kind", ["decoder", "gemma3"])
@pytest.mark.parametrize("page_size, rows", [(16, 24), (64, 80)])
def test_chunks_steps_and_mixed_batches_match_the_oracle(kind, page_size, rows):
    import torch

    from ironmule_amd.paged import PagedCache, PagedDecoder
    announce("paged decoder", kind, page_size, rows)
    weights = make(kind, 7)
    cache = PagedCache(weights.config, 4, CAPACITY, 30, rows, "cuda", page_size=page_size)
    model = PagedDecoder(weights, cache)
    oracle = Oracle(weights, kind, 4)
    rng = np.random.default_rng(rows)
    prompts = [rng.integers(0, 512, n).tolist() for n in (23, 0, 61, 1)]
    got = model.prefill(prompts)
    assert cache.lengths.tolist() == [23, 0, 61, 1]
    assert torch.isnan(got[1]).all()
    for r in (0, 2, 3):
        check(got[r], *oracle.feed(r, prompts[r]), ("prompt", r))
    for counts in ([1, 1, 1, 1], [1, 17, 0, 5], [0, 0, 1, 0]):
        tokens = [rng.integers(0, 512, n).tolist() for n in counts]
        got = model.extend(tokens, counts)
        assert cache.status.tolist() == [0] * 4
        for r, n in enumerate(counts):
            if n:
                check(got[r], *oracle.feed(r, tokens[r]), (counts, r))
            else:
                assert torch.isnan(got[r]).all()


@pytest.mark.parametrize("kind", ["decoder", "gemma3"])
def test_forks_share_a_prefix_and_part(kind):
    import torch

    from ironmule_amd.paged import PagedCache, PagedDecoder
    announce("paged forks", kind)
    weights = make(kind, 8)
    rng = np.random.default_rng(3)
    prompt = rng.integers(0, 512, 37).tolist()
    tails = [rng.integers(0, 512, 4).tolist() for _ in range(3)]
    cache = PagedCache(weights.config, 3, CAPACITY, 12, 40, "cuda", page_size=16)
    model = PagedDecoder(weights, cache)
    model.prefill([prompt, [], []])
    cache.fork(0, [1, 2])
    assert int((cache.refs > 0).sum()) == 3 and cache.refs.max().item() == 3
    alone = PagedCache(weights.config, 3, CAPACITY, 12, 120, "cuda", page_size=16)
    apart = PagedDecoder(weights, alone)
    for r in range(3):  # the same calls, each request with pages of its own
        apart.prefill([prompt if i == r else [] for i in range(3)])
    for step in range(4):
        tokens = [[t[step]] for t in tails]
        a, b = model.extend(tokens, [1] * 3), apart.extend(tokens, [1] * 3)
        assert torch.equal(a, b), step
    assert int((cache.refs > 0).sum()) == 2 + 3  # two whole pages shared, one of each request's own
    cache.release([0, 2])
    assert cache.lengths.tolist() == [0, 41, 0] and int((cache.refs > 0).sum()) == 3
    a, b = model.extend([[], [5], []], [0, 1, 0]), apart.extend([[], [5], []], [0, 1, 0])
    assert torch.equal(a[1], b[1])
    cache.release()
    assert not cache.refs.any() and (cache.tables == -1).all()


@pytest.mark.parametrize("kind, ends", [("decoder", False), ("decoder", True), ("gemma3", False), ("gemma3", True)])
def test_beam_search_finds_what_a_search_without_sharing_finds(kind, ends):
    """A search in torch whose beams share nothing: every step takes every beam's prompt and tokens through
    requests of its own again, in launches of the same rows.  Without an end the logits are the same bits;
    with one the finished beams are missing from the earlier launches, whose sums may round otherwise.
    The scores are held against the oracle's for the same tokens too: a log probability of logits that are
    off by 2 d is off by 4 d at most."""
    import torch

    from ironmule_amd.paged import PagedCache, PagedDecoder
    announce("beam search", kind, ends)
    weights = make(kind, 9)
    beams, steps, groups = 3, 5, 2
    rng = np.random.default_rng(11)
    prompts = [rng.integers(0, 512, n).tolist() for n in (19, 33)]
    cache = PagedCache(weights.config, groups * beams, CAPACITY, 40, 64, "cuda", page_size=16)
    model = PagedDecoder(weights, cache)
    twin = PagedDecoder(weights, PagedCache(weights.config, groups * beams, CAPACITY, 40, 64, "cuda", page_size=16))

    def logits_of(live):
        twin.cache.release()
        for j in range(beams):
            out = twin.prefill([prompts[r // beams] if r % beams == j else [] for r in range(groups * beams)])
            first = out if j == 0 else torch.where(torch.isnan(out), first, out)
        for step in range(max(len(t) for _, t, ended in live if not ended) if live[0][1] else 0):
            first = twin.extend([[] if ended else [t[step]] for _, t, ended in live], [int(not ended) for _, _, ended in live])
        return first.double().log_softmax(1).cpu().numpy()

    live = [(0.0, [], False)] * (groups * beams)
    eos = -1
    for step in range(steps):
        if all(ended for _, _, ended in live):
            break
        logits = logits_of(live)
        if ends and step == 0:
            eos = int(np.argsort(logits[0])[-2])  # the first prompt's second choice: that beam ends at once
        made = []
        for g in range(groups):
            options = []
            for b in range(g * beams, (g + 1) * beams if step else g * beams + 1):
                score, tokens, ended = live[b]
                if ended:
                    options.append((score, tokens + [eos], True))
                else:
                    options += [(score + logits[b, v], tokens + [int(v)], v == eos) for v in np.argsort(-logits[b])[:beams]]
            made += sorted(options, key=lambda o: -o[0])[:beams]
        live = made
    assert any(ended for _, _, ended in live) == ends
    oracle = Oracle(weights, kind, 1)
    for _ in range(2):  # the second search finds the first one's requests in the cache
        tokens, scores = model.beam_search(prompts, beams, steps, eos=eos)
        for i, (score, want, _) in enumerate(live):
            assert tokens[i // beams, i % beams].tolist() == want + [eos] * (steps - len(want)), i
            # the sum of `steps` fp32 log probabilities of size up to 16
            if not ends:
                assert abs(scores.view(-1)[i].item() - score) <= steps * 16 * 2 ** -23
    for i, (_, want, _) in enumerate(live):
        oracle.at[0] = 0
        ref, d = oracle.feed(0, prompts[i // beams])
        score, bound = 0.0, 1e-5
        for token in want:
            score += ref[token] - ref.max() - np.log(np.exp(ref - ref.max()).sum())
            bound += 4 * d
            if token == eos:
                break
            ref, d = oracle.feed(0, [token])
        assert abs(scores.view(-1)[i].item() - score) <= bound, i


def test_a_captured_step_and_one_on_another_stream_give_the_eager_logits():
    import torch

    from ironmule_amd.paged import PagedCache, PagedDecoder
    announce("captured paged step")
    weights = make("decoder", 10)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, 512, n).tolist() for n in (15, 40, 3, 31, 8)]
    caches = [PagedCache(weights.config, 5, CAPACITY, 40, 97, "cuda", page_size=16) for _ in range(3)]
    models = [PagedDecoder(weights, c) for c in caches]
    for m in models:
        m.prefill(prompts)
    tokens, counts = torch.zeros((5, 1), dtype=torch.int32, device="cuda"), torch.ones(5, dtype=torch.int32, device="cuda")
    kept = [c.clone() for c in (caches[0].tables, caches[0].lengths, caches[0].refs)]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = models[0].extend(tokens, counts)
    assert all(torch.equal(a, b) for a, b in zip(kept, (caches[0].tables, caches[0].lengths, caches[0].refs)))
    side = torch.cuda.Stream()
    for step in range(6):
        tokens.copy_(torch.from_numpy(rng.integers(0, 512, (5, 1)).astype(np.int32)))
        if step == 3:
            counts[2] = 0
        graph.replay()
        eager = models[1].extend(tokens, counts)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = models[2].extend(tokens, counts)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(captured.nan_to_num(9.0), eager.nan_to_num(9.0)), step
        assert torch.equal(other.nan_to_num(9.0), eager.nan_to_num(9.0)), step
        assert torch.isnan(eager[2]).all() == (step >= 3)
    assert caches[0].lengths.tolist() == caches[1].lengths.tolist() == [21, 46, 6, 37, 14]


def test_two_graphs_of_two_caches_replayed_at_once():
    import torch

    from ironmule_amd.paged import PagedCache, PagedDecoder
    announce("two captured paged steps at once")
    weights = make("decoder", 12)
    rng = np.random.default_rng(5)
    prompts = [[rng.integers(0, 512, n).tolist() for n in lengths] for lengths in ((15, 40, 3, 31), (60, 2, 9, 33))]
    tokens = torch.from_numpy(rng.integers(0, 512, (4, 1)).astype(np.int32)).cuda()
    counts = torch.ones(4, dtype=torch.int32, device="cuda")
    models = [PagedDecoder(weights, PagedCache(weights.config, 4, CAPACITY, 40, 97, "cuda", page_size=16)) for _ in range(4)]
    for i, m in enumerate(models):
        m.prefill(prompts[i % 2])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for m in models[:2]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(m.extend(tokens, counts))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for step in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for out, m in zip(outs, models[2:]):
            assert torch.equal(out, m.extend(tokens, counts)), step
        torch.cuda.synchronize()


def test_requests_that_do_not_fit_are_left_as_they_were():
    import torch

    from ironmule_amd.paged import PagedCache, PagedDecoder
    announce("paged refusals")
    weights = make("decoder", 13)
    rng = np.random.default_rng(6)
    cache = PagedCache(weights.config, 3, 64, 5, 64, "cuda", page_size=16)
    model = PagedDecoder(weights, cache)
    model.prefill([rng.integers(0, 512, n).tolist() for n in (16, 16, 14)])
    twin = PagedDecoder(weights, PagedCache(weights.config, 3, 64, 12, 64, "cuda", page_size=16))
    rng = np.random.default_rng(6)
    twin.prefill([rng.integers(0, 512, n).tolist() for n in (16, 16, 14)])
    tokens = [[1] * 17, [2] * 33, [3, 4]]  # two pages, three (refused), none
    got = model.extend(tokens, [17, 33, 2])
    assert cache.status.tolist() == [0, 1, 0] and cache.lengths.tolist() == [33, 16, 16]
    want = twin.extend([tokens[0], [], tokens[2]], [17, 0, 2])
    assert torch.isnan(got[1]).all() and torch.isnan(want[1]).all()
    # other rows to a launch, so other orders of sums: the same logits to their roundings (those of ten
    # steps to bf16 a layer and two layers, at most half a step each way)
    for r in (0, 2):
        assert (got[r] - want[r]).abs().max() <= 2 * 20 * 2 ** -8 * want[r].abs().max()
    with pytest.raises(RuntimeError):
        model.prefill([[], [5] * 40, []])
    with pytest.raises(RuntimeError):
        PagedDecoder(weights, PagedCache(weights.config, 3, 16, 5, 64, "cuda", page_size=16)).prefill([[1] * 17, [], []])
    with pytest.raises(RuntimeError):
        model.beam_search([[1] * 60], 3, 8)
    with pytest.raises(ValueError):
        model.extend([[1], [], []], [2, 0, 0])
    with pytest.raises(ValueError):
        model.extend([[1], [1, 2], []], [2, 2, 0])  # within the width, but more than request 0's tokens
    with pytest.raises(ValueError):
        model.extend(torch.zeros((3, 1), dtype=torch.int32), [1, 1, 1])  # on the host
    with pytest.raises(ValueError):
        model.extend([[1] * 65, [], []], [65, 0, 0])
    with pytest.raises(ValueError):
        model.extend(torch.zeros((2, 1), dtype=torch.int32, device="cuda"), [1, 1])
    with pytest.raises(ValueError):
        model.beam_search([[1], [2]], 2, 3)
    with pytest.raises(ValueError):
        model.beam_search([[]], 3, 3)
    with pytest.raises(ValueError):
        PagedDecoder(make("gemma3", 1), cache)
