"""Paged attention with bounds that have to be clipped, value by value, and the paged write beside the slot
path's kernel, each value that differs within the steps that it can differ by."""

from __future__ import annotations

import pytest

from tests.conftest import gpu_available
from tests.gpu_util import announce
from tests.paged_model import attention
from tests.test_paged_gpu import _Batch, _gen

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]


@pytest.fixture(scope="module")
def env():
    import torch

    from ironmule_amd import _native
    code, arch, _ = _native.device_check()
    assert code == 0, f"device {arch} is not supported"
    return torch, _native


@pytest.mark.parametrize("room", [0, 9000])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("last", [20, 900])
def test_starts_and_ends_are_taken_as_the_nearest_bound(env, last, dim, room):
    """Starts before the first row and past the last one, ends past the tables and before 0: what the kernel does
    is what the definition says for the clipped values, and rows of no request stay."""
    torch, n_ = env
    announce("paged attention, clipped", last, dim, room)
    b = _Batch(torch, [(1, 100), (20, 120), (1, 40), (3, 3)], 8, 2, dim, 16, seed=2, room=room)
    b.k.nan_to_num_(0.25)
    b.v.nan_to_num_(-0.5)
    rows, held = b.q.shape[0], b.tables.shape[1] * 16
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    b.starts.copy_(ints(-3, 1, 1, 2, last))
    for ends in ((50, 2**31 - 1, 30, 2**30), (-9, 5, 0, held), (1, 0, 2**31 - 1, 33)):
        b.ends.copy_(ints(*ends))
        before = b.out.clone()
        b.run(n_)
        starts, clipped = ints(0, 1, 1, 2, min(last, rows)), b.ends.clamp(0, held)
        want, bound = attention(torch, b.q, b.k, b.v, b.tables, starts, clipped.clamp(min=1), b.scale)
        for r in (clipped == 0).nonzero()[:, 0].tolist():  # (the model takes no empty request: its rows see nothing)
            want[starts[r]:starts[r + 1]] = 0.0
        there = torch.arange(rows, device="cuda") < starts[-1]
        assert torch.equal(b.out[~there], before[~there])
        assert ((b.out.double() - want).abs() <= bound)[there].all()


def test_a_write_differs_from_the_decode_kernel_by_roundings_only(env):
    """The two add a head's squares in different orders and may have the last bit of an angle otherwise, so a
    normed value may round to its neighbour, 2^-7 of it away, as may the turned one: with len the length of
    the turning pair, 2^-7 (sqrt(2) len + the value) and 2^-22 len for the angle, and in few places."""
    torch, n_ = env
    announce("paged write, decode kernel")
    gen = _gen(torch, 3)
    rows, hq, hkv, cap = 40, 32, 8, 64
    q, k, v = (torch.randn((rows, h, 128), device="cuda", generator=gen).to(torch.bfloat16) for h in (hq, hkv, hkv))
    norms = [torch.empty(128, device="cuda").uniform_(0.9, 1.1, generator=gen).to(torch.bfloat16) for _ in range(2)]
    positions = torch.randint(0, cap, (rows,), dtype=torch.int32, device="cuda", generator=gen)
    slots = torch.arange(rows, dtype=torch.int32, device="cuda")
    pools = [torch.zeros((rows, hkv, cap, 128), dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    one, two = torch.empty_like(q), torch.empty_like(q)
    n_.qk_norm_rope(q, k, v, *norms, positions, slots, one, *pools[:2], 1e6, 1e-6)
    n_.paged_write(q, k, v, *norms, positions, slots * cap + positions, two, *pools[2:], 1e6, 1e-6)
    assert torch.equal(pools[1], pools[3])
    for a, b in ((one, two), (pools[0], pools[2])):
        a, b = a.double(), b.double()
        length = a.unflatten(-1, (2, 64)).square().sum(-2, keepdim=True).sqrt().expand(*a.shape[:-1], 2, 64).flatten(-2)
        assert ((a - b).abs() <= 2.0**-7 * (2**0.5 * length + a.abs()) + 2.0**-22 * length).all()
        assert float((a != b).double().mean()) < 0.01


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("requests", [[(1, 900)], [(1, 9000), (3, 500)], [(200, 900), (1, 600)]])
def test_an_infinite_value_stays_infinite(env, requests, dim):
    """Values of one sign in a dimension, some infinite, at positions that every row sees and that some see: the
    rows that see one have that infinity there and no NaN, the others what the finite values give."""
    torch, n_ = env
    announce("paged attention, infinite values", dim, requests)
    b = _Batch(torch, requests, 8, 2, dim, 16, seed=3)
    for position, at, value in ((5, 0, 1), (70, 9, -1), (131, 9, -1), (300, dim - 1, 1), (requests[0][1] - 1, 40, 1),
                                (requests[0][1] - 150, 77, -1)):
        b.v[int(b.tables[0, position // 16]), :, position % 16, at] = value * float("inf")
    b.run(n_)
    want, bound = attention(torch, b.q, b.k, b.v, b.tables, b.starts, b.ends, b.scale)
    rows = int(b.starts[-1])
    got, want, bound = b.out[:rows].double(), want[:rows], bound[:rows]
    odd = ~want.isfinite()
    assert odd.any() and not want.isnan().any()
    assert torch.equal(got[odd], want[odd])
    assert ((got - want).abs() <= bound)[~odd].all()
