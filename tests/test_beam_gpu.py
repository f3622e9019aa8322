"""GPU parity of beam selection (imq_beam_select) against 64 bits: parents, tokens and flags equal, scores to
fp32's rounding of the key (the log sum's own error, of fp32 exponentials summed in double, is under 2^-24 of
its terms and far below it: 2^-20 of the key's parts bounds both)."""

from __future__ import annotations

import numpy as np
import pytest

from tests.conftest import gpu_available
from tests.gpu_util import announce

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]


@pytest.fixture(scope="module")
def env():
    import torch

    from ironmule_amd import _native
    code, arch, _ = _native.device_check()
    assert code == 0, f"device {arch} is not supported"
    return torch, _native


def _want(logits, scores, beams, count, finished, eos):
    """(scores, parents, tokens, flags) in float64, ties to the lowest (beam, token)."""
    x = logits.double().cpu().numpy()
    rows, vocab = x.shape
    with np.errstate(all="ignore"):
        most = x.max(-1, keepdims=True)
        lse = most + np.log(np.exp(x - most).sum(-1, keepdims=True))
        key = scores.double().cpu().numpy()[:, None] + (x - lse)
    off = ~np.isfinite(lse[:, 0]) | ~np.isfinite(scores.cpu().numpy())
    key[off] = -np.inf
    key[np.isnan(key)] = -np.inf
    if finished is not None:
        for row in np.flatnonzero(finished.cpu().numpy()):
            key[row] = -np.inf
            if np.isfinite(float(scores[row])):
                key[row, eos] = float(scores[row])
    out = []
    for g in range(rows // beams):
        flat = key[g * beams:(g + 1) * beams].reshape(-1)
        best = np.argsort(-flat, kind="stable")[:count]
        for at in best:
            if flat[at] == -np.inf:
                out.append((-np.inf, -1, -1, 0))
            else:
                row, token = g * beams + int(at) // vocab, int(at) % vocab
                done = finished is not None and bool(finished[row])
                out.append((flat[at], row, token, int(done or token == eos)))
        out += [(-np.inf, -1, -1, 0)] * (count - len(best))
    return [np.array(c).reshape(rows // beams, count) for c in zip(*out)]


def _check(torch, n_, logits, scores, beams, count, finished=None, eos=-1):
    got = [t.cpu().numpy() for t in n_.beam_select(logits, scores, beams, count, finished=finished, eos=eos)]
    want = _want(logits, scores, beams, count, finished, eos)
    for g, w in zip(got[1:], want[1:]):
        assert np.array_equal(g, w), (g, w)
    dead = want[1] < 0
    assert np.isneginf(got[0][dead]).all()
    size = 1.0 + np.abs(want[0][~dead]) + float(logits.float().nan_to_num(0.0, 0.0, 0.0).abs().max())
    assert (np.abs(got[0][~dead] - want[0][~dead]) <= 2.0**-20 * size).all()
    return got


@pytest.mark.parametrize("groups,beams,vocab,count,dtype", [
    (1, 1, 1, 1, "float32"), (1, 1, 50, 64, "float32"), (3, 2, 7, 16, "float32"), (1, 4, 151936, 4, "float32"),
    (2, 8, 4096, 16, "float32"), (2, 3, 4097, 6, "bfloat16"), (1, 64, 1000, 64, "float32"), (40, 1, 8191, 3, "bfloat16"),
    (4, 8, 32001, 16, "bfloat16"), (1, 5, 262144, 10, "bfloat16"), (2, 16, 20000, 32, "float32")])
def test_selection_against_64_bits(env, groups, beams, vocab, count, dtype):
    torch, n_ = env
    announce("beam select", groups, beams, vocab, count, dtype)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(vocab + beams)
    rows = groups * beams
    logits = (4.0 * torch.randn((rows, vocab), device="cuda", generator=gen)).to(getattr(torch, dtype))
    scores = -5.0 * torch.rand(rows, device="cuda", generator=gen)
    _check(torch, n_, logits, scores, beams, count)
    if vocab > 2:
        finished = (torch.rand(rows, device="cuda", generator=gen) < 0.4).int() * 3
        _check(torch, n_, logits, scores, beams, count, finished, eos=2)
        # the first step: one beam of each group in use
        scores = torch.full((rows,), float("-inf"), device="cuda")
        scores[::beams] = 0.0
        _check(torch, n_, logits, scores, beams, count, torch.zeros_like(finished), eos=vocab - 1)


def test_ties_go_to_the_lowest(env):
    """Rows of one value, of a few values, of zeros of both signs."""
    torch, n_ = env
    announce("beam select, ties")
    for vocab in (5, 4096, 10000):
        scores = torch.zeros(4, device="cuda")
        _check(torch, n_, torch.full((4, vocab), 1.5, device="cuda"), scores, 2, 12)
        gen = torch.Generator(device="cuda")
        gen.manual_seed(vocab)
        few = torch.randint(0, 3, (4, vocab), device="cuda", generator=gen).float()
        few[1] = few[0]
        few[3] = few[2]
        _check(torch, n_, few, scores, 2, 40)
        signs = torch.zeros((4, vocab), device="cuda")
        signs[:, ::2] = -0.0
        _check(torch, n_, signs.to(torch.bfloat16), scores, 4, 9)


def test_masked_and_broken_logits(env):
    """-inf tokens are never taken; a row of -inf, with a NaN or with +inf offers nothing; scores that are not finite
    neither; fewer continuations than asked for end in -inf, -1, -1, 0."""
    torch, n_ = env
    announce("beam select, not finite")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    inf, nan = float("inf"), float("nan")
    logits = torch.randn((10, 9000), device="cuda", generator=gen)
    logits[0, 5:] = -inf
    logits[1] = -inf
    logits[2, 8000] = nan
    logits[3, 17] = inf
    logits[4, :8999] = -inf
    logits[6, 4096:] = -inf
    scores = torch.randn(10, device="cuda", generator=gen)
    scores[5], scores[7], scores[8] = nan, inf, -inf
    _check(torch, n_, logits, scores, 5, 20)
    _check(torch, n_, logits, scores, 1, 8)
    _check(torch, n_, logits, scores, 10, 64, (scores > 0).int(), eos=3)


def test_rows_of_a_wider_matrix(env):
    torch, n_ = env
    announce("beam select, strided")
    wide = torch.randn((6, 5003), device="cuda")
    _check(torch, n_, wide[:, :4999], torch.randn(6, device="cuda"), 3, 6)
    _check(torch, n_, wide.to(torch.bfloat16)[::2, 1:4000], torch.randn(3, device="cuda"), 3, 6)


def test_refusals_on_the_gpu(env):
    torch, n_ = env
    announce("beam select, refusals")
    logits, scores = torch.zeros((4, 100), device="cuda"), torch.zeros(4, device="cuda")
    for args, kw in (((logits, scores, 2, 65), {}), ((logits, scores, 2, 0), {}),
                     ((logits, scores, 2, 2), dict(finished=torch.zeros(4, dtype=torch.int32, device="cuda"), eos=100))):
        with pytest.raises(n_.NativeError):
            n_.beam_select(*args, **kw)
    with pytest.raises(ValueError):
        n_.beam_select(logits, scores.cpu(), 2, 2)
