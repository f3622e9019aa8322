"""The probabilities of steps and short chunks over pages are two terms of bf16 for the product with the values, as
those of the slots' decode attention are: values of both signs that all but cancel show what is lost."""

from __future__ import annotations

import pytest

from tests.conftest import gpu_available
from tests.gpu_util import announce
from tests.paged_model import attention
from tests.test_paged_gpu import _Batch, _gen

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]

DELTA = 0.6875             # exp(-DELTA) = 0.50283, which bf16 has as 129 / 256
WEIGHT = 129 / 256


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("requests", [
    [(1, 40)], [(1, 777)], [(1, 8000)], [(1, 100 + 61 * i) for i in range(40)], [(8, 300), (1, 2000)], [(3, 3), (2, 1500)],
    [(1, 900), (300, 300), (8, 64)]])
def test_sums_that_cancel(dim, requests):
    """Every other key scores DELTA less and its values are the others' over -WEIGHT: the output is a thousandth of
    the values, and nothing if the probability is rounded to bf16.  The first term has a probability's upper eight
    bits, cut off: less than 2^-7 of it is left (8 bits, the first one 1), of which the second term's rounding
    takes half a step, 2^-8 of that at most: 2^-15.  The 2^-20 that is added scales the whole output (2^-20 of it,
    within its rounding's 2^-8).  The rest of the bound as in paged_model.attention, of values up to 1."""
    import torch

    from ironmule_amd import _native
    announce("paged attention, cancelling", dim, requests)
    b = _Batch(torch, requests, 8, 2, dim, 16, seed=1)
    gen = _gen(torch, 7)
    sign = 1.0 - 2.0 * torch.randint(0, 2, (dim,), device="cuda", generator=gen).float()
    b.q.zero_()
    b.q[..., 0] = 1.0
    for pool in (b.k, b.v):
        pool.zero_()
    b.k[:, :, 1::2, 0] = -DELTA  # (a page holds an even number of tokens)
    b.v[:, :, 0::2] = (-WEIGHT * sign).to(torch.bfloat16)
    b.v[:, :, 1::2] = sign.to(torch.bfloat16)
    b.scale = 1.0
    b.run(_native)
    want, _ = attention(torch, b.q, b.k, b.v, b.tables, b.starts, b.ends, 1.0)
    u, longest = 2.0 ** -24, max(end for _, end in requests)
    rest = 2.0 ** -15 + 2 * (dim + 8) * u * DELTA + 2 * (longest / 16 + 64) * u
    starts = b.starts.tolist()
    for r, (n, _) in enumerate(requests):
        if 4 * n > 32:
            continue  # (tiles of many queries: one term)
        got, ref = b.out[starts[r]:starts[r + 1]].double(), want[starts[r]:starts[r + 1]]
        off = (got - ref).abs()
        print("[cancelling]", requests[r], f"{float(off.max()):.2e} of {rest:.2e}", flush=True)
        assert (off <= 2.0 ** -8 * ref.abs() + rest).all()
