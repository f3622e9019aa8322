"""Scores of beam selection (imq_beam_select) to fp32's rounding of the key, whatever the size of the logits:
rows with a large common offset, peaked rows, tokens masked with the lowest finite value, rows of nothing else.

The bar, with u = 2^-24 and t = (largest logit) - (a logit): a term of the sum is exp2 of t log2(e), whose argument
has three roundings (the difference, log2(e), their product), 3 u t of it, and exp2 itself is good to one
unit in the last place, 2 u; eight terms are added in fp32, 7 u; everything else is in double.  The log of the sum
is then off by at most u (3 mean(t) + 9), the mean weighted by the probabilities, and by as much again and 2 u
for each further block of 4096 values that one wavefront takes (rows there are 2048 of).  The score's own rounding: u of it.
"""

from __future__ import annotations

import numpy as np
import pytest

from tests.conftest import gpu_available
from tests.gpu_util import announce

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]

U = 2.0 ** -24
FLOAT_MIN, BF16_MIN = -float(np.finfo(np.float32).max), -3.3895313892515355e38


@pytest.fixture(scope="module")
def env():
    import torch

    from ironmule_amd import _native
    code, arch, _ = _native.device_check()
    assert code == 0, f"device {arch} is not supported"
    return torch, _native


def _check(env, logits, scores, beams, count, blocks=1, finished=None, eos=-1):
    """Every output of a call against 64 bits: keys (x - most) - log(sum exp(x - most)) + score, ties to the lowest."""
    torch, n_ = env
    got = [t.cpu().numpy() for t in n_.beam_select(logits, scores, beams, count, finished=finished, eos=eos)]
    x, score = logits.double().cpu().numpy(), scores.double().cpu().numpy()
    rows, vocab = x.shape
    most = x.max(-1, keepdims=True)
    weight = np.exp(x - most)
    sums = weight.sum(-1, keepdims=True)
    key = score[:, None] + ((x - most) - np.log(sums))
    mean = (weight * np.where(weight > 0, most - x, 0.0)).sum(-1) / sums[:, 0]
    bound = U * (3 * mean + 9 + (blocks - 1) * (3 * mean + 2))
    if finished is not None:
        for row in np.flatnonzero(finished.cpu().numpy()):
            key[row], key[row, eos], bound[row] = -np.inf, score[row], 0.0
    for g in range(rows // beams):
        flat = key[g * beams:(g + 1) * beams].reshape(-1)
        best = np.argsort(-flat, kind="stable")[:count]
        best = best[flat[best] > -np.inf]
        n, row, token = len(best), g * beams + best // vocab, best % vocab
        assert np.array_equal(got[1][g, :n], row) and np.array_equal(got[2][g, :n], token), (g, got[1][g], row, got[2][g], token)
        assert (got[1][g, n:] == -1).all() and np.isneginf(got[0][g, n:]).all()
        off = np.abs(got[0][g, :n] - flat[best])
        assert (off <= bound[row] + U * np.abs(flat[best])).all(), (g, got[0][g, :n], flat[best], off / bound[row])


def _normal(torch, rows, vocab, seed, scale=3.0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return scale * torch.randn((rows, vocab), device="cuda", generator=gen)


@pytest.mark.parametrize("offset", [0.0, 300.0, -3000.0, 30000.0])
@pytest.mark.parametrize("rows,vocab,blocks", [(4, 8192, 1), (6, 151936, 1), (2048, 9001, 3)])
def test_a_common_offset_leaves_the_scores(env, offset, rows, vocab, blocks):
    torch, _ = env
    announce("beam scores, offset", offset, rows, vocab)
    logits = _normal(torch, rows, vocab, vocab) + offset * (1.0 + 0.01 * torch.arange(rows, device="cuda")[:, None] / rows)
    _check(env, logits, torch.zeros(rows, device="cuda"), 1 if rows > 100 else 2, 6, blocks)


@pytest.mark.parametrize("peak", [42.0, 301.0, 3003.0, 3e7])
def test_a_peaked_row_scores_zero(env, peak):
    """One logit far above the others: its log probability is 0 or a little below, never above."""
    torch, n_ = env
    announce("beam scores, peaked", peak)
    logits = _normal(torch, 4, 20000, 5)
    logits[torch.arange(4), torch.tensor([3, 7000, 12345, 19999])] = peak * torch.tensor([1.0, 0.9, 1.1, 0.7], device="cuda")
    _check(env, logits, torch.zeros(4, device="cuda"), 1, 3)
    scores = n_.beam_select(logits, torch.zeros(4, device="cuda"), 1, 1)[0]
    assert (scores <= 0).all()  # (the largest logit's own term is 1)


@pytest.mark.parametrize("dtype,lowest", [("float32", FLOAT_MIN), ("bfloat16", BF16_MIN)])
@pytest.mark.parametrize("rows,blocks", [(4, 1), (2048, 3)])
def test_tokens_masked_with_the_lowest_finite_value(env, dtype, lowest, rows, blocks):
    """Few tokens allowed, anywhere; whole wavefronts of masked ones before and behind them; nothing but masked
    ones; masks of the lowest value and of -inf side by side; and logits near the largest value."""
    torch, _ = env
    announce("beam scores, lowest finite", dtype, rows)
    vocab, kind = 9000, getattr(torch, dtype)
    logits = torch.full((rows, vocab), lowest, device="cuda", dtype=kind)
    assert float(logits[0, 0]) == lowest
    some = torch.arange(5, device="cuda")
    logits[0::4, :5] = some.to(kind)
    logits[1::4, 8990:8995] = (some - 40).to(kind)
    logits[2::4, 4500:4505] = (7.5 * some).to(kind)
    scores = -0.3 * torch.arange(rows, device="cuda").float().remainder(4)
    _check(env, logits, scores, 4, 7, blocks)     # (rows 3, 7, ..: masked as a whole)
    _check(env, logits, scores, 1, 9, blocks)     # more continuations than there are allowed tokens
    logits[0::4, 100:] = float("-inf")
    logits[3::4, :8999] = float("-inf")
    _check(env, logits, scores, 4, 24, blocks)
    high = _normal(torch, rows, vocab, 3).to(kind)
    high[:, 1000:5000] = 3e38
    high[1::2, 4999] = 3.2e38
    _check(env, high, scores, 2, 6, blocks)


def test_finished_beams_beside_masked_ones(env):
    torch, _ = env
    announce("beam scores, finished and masked")
    logits = torch.full((6, 5000), FLOAT_MIN, device="cuda")
    logits[0, 17], logits[3, 4000] = 1.0, -2.0
    finished = torch.tensor([0, 1, 0, 0, 0, 1], dtype=torch.int32, device="cuda")
    _check(env, logits, torch.tensor([-3.0, -1.0, -2.0, -0.5, -9.0, -20.0], device="cuda"), 3, 6, finished=finished, eos=2)
