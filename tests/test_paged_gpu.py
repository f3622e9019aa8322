"""GPU parity of the paged cache (include/ironmule_paged.h): pages shared out and reordered against the
plain model, value by value; norm and rotary into pages, and attention over pages, against 64 bits.

Bars: tables, rows, slots and copied pages equal.  A written head differs from the 64-bit one by the two
bf16 roundings it takes (after the norm and after the rotation), 2^-8 each of the turning pair's
length, and fp32 arithmetic, 2^-20 of it.  Attention: the bound of tests/paged_model.py.
"""

from __future__ import annotations

import numpy as np
import pytest

from tests.conftest import gpu_available
from tests.gpu_util import announce
from tests.paged_model import PagedModel, attention

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]


@pytest.fixture(scope="module")
def env():
    import torch

    from ironmule_amd import _native
    code, arch, _ = _native.device_check()
    assert code == 0, f"device {arch} is not supported"
    return torch, _native


def _gen(torch, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


# ------------------------------------------------------------------ tables

class _Device:
    """A cache's arrays and a chunk's on the GPU, next to the model."""

    def __init__(self, torch, n_, model, rows, planes=0, inner=(2, 16, 8)):
        self.torch, self.n_, self.model, self.rows = torch, n_, model, rows
        put = lambda a: torch.from_numpy(a.copy()).cuda()  # noqa: E731
        self.tables, self.lengths, self.refs = put(model.tables), put(model.lengths), put(model.refs)
        requests = model.tables.shape[0]
        ints = lambda *s: torch.full(s, -7, dtype=torch.int32, device="cuda")  # noqa: E731
        self.chunk = dict(starts=ints(requests + 1), ends=ints(requests), status=ints(requests), positions=ints(rows),
                          slots=ints(rows), copies=ints(requests, 2))
        self.pool = None
        if planes:
            self.pool = torch.randint(-2**15, 2**15, (planes, len(model.refs), *inner), dtype=torch.int16, device="cuda")

    def cache(self):
        return self.tables, self.lengths, self.refs

    def reserve(self, counts):
        torch, want_pool = self.torch, None
        if self.chunk["positions"].numel() != self.rows:
            for name in ("positions", "slots"):
                self.chunk[name] = self.torch.full((self.rows,), -7, dtype=self.torch.int32, device="cuda")
        want = self.model.reserve(counts, self.rows)
        if self.pool is not None:
            want_pool = self.pool.clone()
            for old, new in want["copies"]:
                if old >= 0:
                    want_pool[:, new] = self.pool[:, old]
        self.n_.paged_reserve(*self.cache(), torch.from_numpy(np.asarray(counts, np.int32)).cuda(), self.model.page,
                              **self.chunk, pool=self.pool)
        self.agree()
        for name, value in want.items():
            got = self.chunk[name].cpu().numpy()
            assert np.array_equal(got, value), (name, got, value)
        if self.pool is not None:
            assert torch.equal(self.pool, want_pool)
        return want

    def reorder(self, parents):
        self.model.reorder(parents)
        self.n_.paged_reorder(*self.cache(), self.torch.from_numpy(np.asarray(parents, np.int32)).cuda(), self.model.page)
        self.agree()

    def agree(self):
        for name in ("tables", "lengths", "refs"):
            got, want = getattr(self, name).cpu().numpy(), getattr(self.model, name)
            assert np.array_equal(got, want), (name, got, want)

    def commit(self):
        self.lengths.copy_(self.chunk["ends"])
        self.model.lengths = self.chunk["ends"].cpu().numpy().copy()


@pytest.mark.parametrize("requests,columns,pages,page,rows,most", [
    (1, 1, 1, 16, 20, 24), (5, 9, 30, 16, 120, 60), (33, 7, 100, 64, 700, 90), (3, 40, 37, 32, 1500, 700),
    (1024, 3, 1500, 16, 4000, 9), (200, 130, 9000, 16, 30000, 400)])
def test_rounds_of_a_cache_agree_with_the_model(env, requests, columns, pages, page, rows, most):
    """Random rounds: reservations (too large ones, malformed ones, more rows than there are), commits of all or
    of a part, forks, ends, and parents that do not exist."""
    torch, n_ = env
    announce("paged rounds", requests, columns, pages, page)
    rng = np.random.default_rng(requests * 1000 + columns)
    device = _Device(torch, n_, PagedModel(requests, columns, pages, page), rows, planes=3)
    seen = set()
    for _ in range(25):
        if rng.random() < 0.4:
            parents = np.arange(requests)
            some = rng.random(requests) < 0.4
            parents[some] = rng.integers(-2, requests + 1, int(some.sum()))
            device.reorder(parents)
        else:
            counts = rng.integers(0, most + 1, requests) * (rng.random(requests) < 0.6)
            counts[rng.random(requests) < 0.02] = -1
            seen |= set(device.reserve(counts)["status"].tolist())
            if rng.random() < 0.7:
                device.commit()
                if rng.random() < 0.3:  # only some of the new tokens are kept
                    least = device.model.lengths // page * page
                    device.model.lengths = np.maximum(least, device.model.lengths - 1).astype(np.int32)
                    device.lengths.copy_(torch.from_numpy(device.model.lengths))
        device.model.check()
    print("[statuses]", sorted(seen))


def test_more_pages_than_one_list_holds(env):
    """Some 60000 pages in one call, more than twice what is listed at a time; then calls for more than are left,
    with requests refused in the middle of a list and behind it."""
    torch, n_ = env
    announce("paged reserve, long lists")
    device = _Device(torch, n_, PagedModel(5, 30000, 100003, 16), 1 << 20)
    device.reserve([19000 * 16, 1, 22000 * 16 - 3, 0, 19000 * 16])
    device.commit()
    device.reorder([0, 1, 2, 1, 4])
    device.reserve([11000 * 16, 29999 * 16 - 5, 5, 12000 * 16, 1])
    device.commit()
    device.reorder([-1, 0, 2, -1, 4])
    device.reorder([0, 1, -1, -1, -1])
    device.rows = 0
    want = device.reserve([30000 * 16] * 2 + [25000 * 16, 30000 * 16, 16])
    assert 0 not in want["status"][2:]


def test_lists_end_where_pages_do(env):
    """Requests that fit the free pages exactly, by one page less and by one more, lists of several lengths."""
    torch, n_ = env
    announce("paged reserve, exact fits")
    for pages in (3, 1000, 24576, 24577, 50000):
        for over in (-1, 0, 1):
            device = _Device(torch, n_, PagedModel(3, 60000, pages, 16), 1 << 20)
            want = device.reserve([(pages // 3) * 16, 0, (pages - pages // 3 + over) * 16])
            assert want["status"].tolist() == [0, 0, int(over > 0)]


def test_a_shared_page_past_the_tokens_is_refused(env):
    """Tokens given up past a whole shared page: what follows must not be written into it."""
    torch, n_ = env
    announce("paged reserve, shared page past the tokens")
    model = PagedModel(3, 6, 20, 16)
    device = _Device(torch, n_, model, 100)
    device.reserve([48, 0, 0])
    device.commit()
    device.reorder([0, 0, -1])
    model.lengths[0] = 10  # pages 1 and 2 are still held, and shared
    device.lengths[0] = 10
    want = device.reserve([30, 3, 20])
    assert want["status"].tolist() == [2, 0, 0]


def test_no_rows_and_nothing_to_do(env):
    torch, n_ = env
    announce("paged reserve, no rows")
    device = _Device(torch, n_, PagedModel(2, 3, 4, 16), 0)
    device.reserve([0, 0])
    assert device.reserve([1, 0])["status"].tolist() == [3, 0]


# ------------------------------------------------------------------ rows into pages

def _wide(torch, rows, heads, dim, extra, gen):
    """(rows, heads, dim) bf16 normal values, rows `extra` values further apart than they are long."""
    width = heads * dim
    return torch.randn((rows, width + extra), device="cuda", generator=gen).to(torch.bfloat16)[:, :width].unflatten(1, (heads, dim))


@pytest.mark.parametrize("rows,heads,kv_heads,dim,page,extra", [
    (1, 32, 8, 128, 16, 0), (7, 16, 8, 256, 64, 64), (300, 5, 5, 128, 32, 8), (65, 7, 1, 256, 128, 0), (33, 1, 1, 128, 1024, 1024)])
def test_write_against_64_bits(env, rows, heads, kv_heads, dim, page, extra):
    torch, n_ = env
    announce("paged write", rows, heads, kv_heads, dim, page, extra)
    gen = _gen(torch, rows)
    q, k, v = (_wide(torch, rows, h, dim, extra, gen) for h in (heads, kv_heads, kv_heads))
    q[0] *= 100.0
    q_norm, k_norm = (torch.empty(dim, device="cuda").uniform_(0.5, 1.5, generator=gen).to(torch.bfloat16) for _ in range(2))
    pages = rows // page + 3
    positions = torch.randint(0, 1 << 20, (rows,), dtype=torch.int32, device="cuda", generator=gen)
    slots = torch.randperm(pages * page, device="cuda", generator=gen)[:rows].to(torch.int32)
    if rows > 5:
        slots[3], slots[rows - 1] = -1, pages * page
    out = _wide(torch, rows, heads, dim, extra, gen)
    pools = [torch.randn((pages, kv_heads, page, dim), device="cuda", generator=gen).to(torch.bfloat16) for _ in range(2)]
    before = [t.clone() for t in (out, *pools)]
    n_.paged_write(q, k, v, q_norm, k_norm, positions, slots, out, *pools, theta=1e6, eps=1e-6)
    angle = positions.double()[:, None] * 1e6 ** (-torch.arange(dim // 2, device="cuda", dtype=torch.float64) * 2 / dim)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]

    def turned(x, weight):
        x = x.double()
        x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * weight.double()
        lo, hi = x[..., :dim // 2], x[..., dim // 2:]
        length = (lo.square() + hi.square()).sqrt()
        return torch.cat([lo * cos - hi * sin, lo * sin + hi * cos], -1), torch.cat([length, length], -1) * (2 * 2.0**-8 + 2.0**-20)

    live = (slots >= 0) & (slots < pages * page)
    want, bound = turned(q, q_norm)
    assert ((out.double() - want).abs() <= bound)[live].all()
    assert torch.equal(out[~live], before[0][~live])
    page_of, offset = slots[live].long() // page, slots[live].long() % page
    want, bound = turned(k, k_norm)
    assert ((pools[0][page_of, :, offset].double() - want[live]).abs() <= bound[live]).all()
    assert torch.equal(pools[1][page_of, :, offset], v[live])
    rest = torch.ones((pages, page), dtype=torch.bool, device="cuda")
    rest[page_of, offset] = False
    for pool, old in zip(pools, before[1:]):
        assert torch.equal(pool.transpose(1, 2)[rest], old.transpose(1, 2)[rest])


def test_write_agrees_with_the_decode_kernel(env):
    """Bit for bit the q and the cache rows of imq_qk_norm_rope (whose angles are computed alike) but where the base,
    there in fp32, is not exact: theta 1e6 is."""
    torch, n_ = env
    announce("paged write and qk_norm_rope")
    gen = _gen(torch, 3)
    rows, hq, hkv, cap = 9, 32, 8, 64
    q, k, v = (torch.randn((rows, h, 128), device="cuda", generator=gen).to(torch.bfloat16) for h in (hq, hkv, hkv))
    norms = [torch.empty(128, device="cuda").uniform_(0.9, 1.1, generator=gen).to(torch.bfloat16) for _ in range(2)]
    positions = torch.randint(0, cap, (rows,), dtype=torch.int32, device="cuda", generator=gen)
    slots = torch.arange(rows, dtype=torch.int32, device="cuda")
    pools = [torch.zeros((rows, hkv, cap, 128), dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    one, two = torch.empty_like(q), torch.empty_like(q)
    n_.qk_norm_rope(q, k, v, *norms, positions, slots, one, *pools[:2], 1e6, 1e-6)
    n_.paged_write(q, k, v, *norms, positions, slots * cap + positions, two, *pools[2:], 1e6, 1e-6)
    differ = float((one != two).float().mean()), float((pools[0] != pools[2]).float().mean())
    print("[differ]", differ)
    assert torch.equal(pools[1], pools[3])
    # the angles may round differently in the last fp32 bit, which moves few values by a bf16 step
    assert max(differ) < 0.01


# ------------------------------------------------------------------ attention

class _Batch:
    def __init__(self, torch, requests, heads, kv_heads, dim, page, seed, extra=0, spare=7, room=0):
        """`requests`: (new tokens, tokens with them) each; pages scattered, what lies past a request's end NaN;
        tables for `room` tokens at least (where little room is left tiles stay whole)."""
        gen = _gen(torch, seed)
        needs = [-(-end // page) for _, end in requests]
        pages = sum(needs) + spare
        order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
        self.tables = torch.full((len(requests), max(max(needs) + 1, room // page)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for r, need in enumerate(needs):
            self.tables[r, :need] = order[at:at + need]
            at += need
        self.k, self.v = (torch.full((pages, kv_heads, page, dim), float("nan"), dtype=torch.bfloat16, device="cuda")
                          for _ in range(2))
        for r, (_, end) in enumerate(requests):
            if end:
                for pool in (self.k, self.v):
                    rows = torch.randn((needs[r] * page, kv_heads, dim), device="cuda", generator=gen).to(torch.bfloat16)
                    rows[end:] = float("nan")
                    pool[self.tables[r, :needs[r]].long()] = rows.unflatten(0, (needs[r], page)).transpose(1, 2)
        counts = [n for n, _ in requests]
        rows = sum(counts)
        self.starts = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device="cuda")
        self.ends = torch.tensor([end for _, end in requests], dtype=torch.int32, device="cuda")
        self.q, self.out = (_wide(torch, rows + 3, heads, dim, extra, gen) for _ in range(2))
        self.scale = dim ** -0.5

    def run(self, n_, window=0, **kw):
        return n_.paged_attention(self.q, self.k, self.v, self.tables, self.starts, self.ends, self.out, self.scale,
                                  window=window, **kw)

    def check(self, torch, n_, window=0, **kw):
        before = self.out.clone()
        self.run(n_, window, **kw)
        want, bound = attention(torch, self.q, self.k, self.v, self.tables, self.starts, self.ends, self.scale, window)
        rows = int(self.starts[-1])
        assert torch.equal(self.out[rows:], before[rows:])  # rows behind the last request
        got, want, bound = self.out[:rows].double(), want[:rows], bound[:rows]
        odd = ~want.isfinite()
        same = torch.equal(got.isfinite(), ~odd)
        assert same, (got.isfinite() == odd).nonzero()[:5]
        ratio = torch.where(odd, 0.0, (got - want).abs() / bound)
        print("[attention]", f"{float(ratio.max()) if ratio.numel() else 0.0:.3f} of the bound", flush=True)
        assert (ratio <= 1.0).all(), (ratio > 1).nonzero()[:5]
        return got


HEADS = [(32, 8, 128), (16, 8, 256), (5, 5, 128), (12, 1, 256), (20, 4, 128)]
BATCHES = [
    [(1, 1)], [(1, 16)], [(1, 17)], [(1, 777)], [(1, 31), (1, 32), (1, 33), (1, 64), (1, 65), (1, 300)],
    [(2, 2), (3, 70), (0, 20), (1, 5), (0, 0)], [(64, 64)], [(65, 1000)], [(129, 129), (1, 500), (33, 64), (7, 7)],
    [(300, 555), (0, 3), (16, 16)],
]


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("batch", range(len(BATCHES)))
@pytest.mark.parametrize("page", [16, 64])
def test_attention_against_64_bits(env, heads, kv_heads, dim, batch, page):
    torch, n_ = env
    announce("paged attention", heads, kv_heads, dim, BATCHES[batch], page)
    _Batch(torch, BATCHES[batch], heads, kv_heads, dim, page, seed=batch).check(torch, n_)


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("batch", range(len(BATCHES)))
def test_attention_with_room_in_the_tables_against_64_bits(env, heads, kv_heads, dim, batch):
    torch, n_ = env
    announce("paged attention, room", heads, kv_heads, dim, BATCHES[batch])
    _Batch(torch, BATCHES[batch], heads, kv_heads, dim, 32, seed=batch + 20, room=9000).check(torch, n_)


@pytest.mark.parametrize("requests,heads,kv_heads,dim", [
    ([(1, 760)], 32, 8, 128), ([(1, 1000)], 32, 8, 128), ([(1, 380)], 16, 8, 256), ([(1, 500)], 16, 8, 256),
    ([(1, 1000 - i) for i in range(4)], 32, 8, 128), ([(1, 2000 - 90 * i) for i in range(16)], 32, 8, 128),
    ([(1, 2040)] * 15, 32, 8, 128), ([(2, 1000 + i) for i in range(20)], 64, 8, 256), ([(4, 1500)] * 70, 16, 2, 128)])
def test_steps_around_the_lengths_that_leave_tiles_whole(env, requests, heads, kv_heads, dim):
    torch, n_ = env
    announce("paged attention, whole or cut", len(requests), requests[0], heads, dim)
    for room in (0, 8192):
        _Batch(torch, requests, heads, kv_heads, dim, 16, seed=11, room=room).check(torch, n_)


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS[:3])
@pytest.mark.parametrize("window", [1, 16, 33, 64, 100, 1024])
def test_windows_against_64_bits(env, heads, kv_heads, dim, window):
    torch, n_ = env
    announce("paged attention, window", heads, kv_heads, dim, window)
    _Batch(torch, [(1, 1), (1, 700), (90, 90), (200, 1300), (1, 64), (17, 400)], heads, kv_heads, dim, 32,
           seed=window).check(torch, n_, window)


@pytest.mark.parametrize("requests,heads,kv_heads,dim,page,extra,window", [
    ([(1, 20000)], 32, 8, 128, 16, 0, 0), ([(1, 9001), (1, 3), (1, 12345)], 16, 8, 256, 64, 64, 0),
    ([(1, 100 + 37 * i) for i in range(48)], 32, 8, 128, 128, 8, 0), ([(700, 5000), (1, 4000)], 8, 2, 128, 1024, 0, 0),
    ([(5, 3000)] * 7, 64, 1, 128, 16, 0, 0), ([(1, 6000), (400, 6000)], 16, 8, 256, 256, 0, 1024),
    ([(600, 600)], 3, 1, 256, 16, 24, 0), ([(1, 5)] * 1024, 2, 1, 128, 16, 0, 0)])
def test_long_and_wide_batches_against_64_bits(env, requests, heads, kv_heads, dim, page, extra, window):
    torch, n_ = env
    announce("paged attention, large", len(requests), requests[0], heads, kv_heads, dim, page, extra, window)
    _Batch(torch, requests, heads, kv_heads, dim, page, seed=5, extra=extra).check(torch, n_, window)


@pytest.mark.parametrize("requests,heads,kv_heads,dim,page,window", [
    # tiles whole, cut for every CU, cut for all that are resident; many of them, few of them, other kinds between
    ([(700, 3000), (220, 1500), (1, 2000)], 16, 8, 256, 16, 512), ([(300, 2500), (300, 2500)], 32, 8, 128, 16, 900),
    ([(512, 2000)], 32, 8, 128, 64, 0), ([(512, 2100)], 32, 8, 128, 64, 0), ([(130, 4100)], 8, 2, 256, 32, 0),
    ([(40, 300)] * 70 + [(1, 900)] * 3, 8, 2, 128, 32, 0), ([(70, 1300 + 10 * i) for i in range(66)], 4, 4, 128, 16, 700),
    ([(33, 5000), (129, 129), (9, 2000)], 32, 1, 128, 16, 0), ([(65, 2048), (1, 2048)], 16, 8, 256, 128, 2000)])
def test_tiles_however_they_are_cut_against_64_bits(env, requests, heads, kv_heads, dim, page, window):
    torch, n_ = env
    announce("paged attention, tiles", len(requests), requests[0], heads, kv_heads, dim, page, window)
    _Batch(torch, requests, heads, kv_heads, dim, page, seed=6).check(torch, n_, window)


@pytest.mark.parametrize("dim", [128, 256])
def test_a_window_that_holds_everything_is_none(env, dim):
    torch, n_ = env
    announce("paged attention, wide windows", dim)
    b = _Batch(torch, [(1, 700), (200, 500), (40, 40)], 8, 2, dim, 16, seed=9)
    want = b.check(torch, n_).clone()
    for window in (b.tables.shape[1] * 16, 1 << 30, 2**31 - 1):
        assert torch.equal(b.check(torch, n_, window), want), window


def test_bounds_on_the_context_change_nothing(env):
    torch, n_ = env
    announce("paged attention, max_context")
    for requests in ([(1, 900), (1, 5), (3, 400)], [(300, 900), (1, 2000)], [(200, 5000)]):
        b = _Batch(torch, requests, 32, 8, 128, 16, seed=8)
        for most in (5000, 1 << 20, 900, 64, 1):  # one that is too small only plans badly
            b.check(torch, n_, max_context=most)
    with pytest.raises(n_.NativeError):
        b.run(n_, max_context=0)


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("requests", [[(1, 200)] * 3, [(150, 200), (40, 40)]])
def test_infinities_and_nans_stay_where_they_are_seen(env, dim, requests):
    """Queries, keys and values of single positions that are not finite: the rows that see them are not finite (in
    the dimensions concerned), every other row is as if they were not there; at the edges of windows too."""
    torch, n_ = env
    announce("paged attention, not finite", dim, requests)
    for window, room in ((0, 0), (50, 0), (0, 9000), (50, 9000)):
        b = _Batch(torch, requests, 8, 2, dim, 16, seed=dim + window, room=room)
        inf, nan = float("inf"), float("nan")
        for pool, position, at, value in ((b.v, 195, 3, inf), (b.v, 160, 7, nan), (b.v, 100, slice(None), -inf),
                                          (b.v, 199, 0, nan), (b.k, 170, 5, nan)):
            pool[int(b.tables[0, position // 16]), :, position % 16, at] = value
        if requests[0][0] == 1:
            b.q[1, 2] = nan
        got = b.check(torch, n_, window)
        assert not got[int(b.starts[0]):int(b.starts[1])].isfinite().all() and got[-1, 0].isfinite().all()


@pytest.mark.parametrize("room", [0, 9000])
def test_bad_table_entries_and_odd_requests(env, room):
    """Pages outside the pool are left out, a request that ends before its rows begin sees nothing, ends past the tables
    and rows past the batch are cut off; nothing outside is read (the host refuses the rest)."""
    torch, n_ = env
    announce("paged attention, bad tables")
    b = _Batch(torch, [(1, 100), (20, 120), (1, 40), (3, 3)], 8, 2, 128, 16, seed=2, room=room)
    pages = b.k.shape[0]
    b.tables[0, 2], b.tables[1, 0], b.tables[1, 7], b.tables[2, :3] = -1, pages, 2**31 - 1, -5
    b.check(torch, n_)
    assert not b.out[21].any()  # every page of it was bad
    b.ends[3] = -4
    b.run(n_)
    assert not b.out[22:25].any()
    b.ends[3] = 1
    b.run(n_)
    assert not b.out[22:24].any() and b.out[24].isfinite().all()
    keep = b.out.clone()
    b.starts.copy_(torch.tensor([-3, 1, 1, 2, 900], dtype=torch.int32))
    b.ends.copy_(torch.tensor([50, 2**31 - 1, 30, 2**30], dtype=torch.int32))
    b.run(n_)
    torch.cuda.synchronize()
    assert b.out.shape == keep.shape


def test_every_row_in_the_same_place_gives_the_same_bits(env):
    torch, n_ = env
    announce("paged attention, twice")
    b = _Batch(torch, [(1, 5000), (300, 4000), (1, 3)], 32, 8, 128, 16, seed=4)
    first = b.run(n_).clone()
    for _ in range(3):
        assert torch.equal(b.run(n_), first)


@pytest.mark.parametrize("rows,heads,kv_heads,dim,extra", [(9, 32, 8, 128, 0), (300, 16, 8, 256, 64)])
def test_a_write_over_its_own_queries(env, rows, heads, kv_heads, dim, extra):
    torch, n_ = env
    announce("paged write in place", rows, heads, dim)
    gen = _gen(torch, rows)
    q, k, v = (_wide(torch, rows, h, dim, extra, gen) for h in (heads, kv_heads, kv_heads))
    weight = torch.ones(dim, device="cuda", dtype=torch.bfloat16)
    positions = torch.arange(rows, dtype=torch.int32, device="cuda")
    slots = positions.clone()
    slots[2] = -1
    apart, over = q.clone(), q
    pools = [torch.zeros((rows // 16 + 1, kv_heads, 16, dim), device="cuda", dtype=torch.bfloat16) for _ in range(4)]
    n_.paged_write(q.clone(), k, v, weight, weight, positions, slots, apart, *pools[:2], theta=1e4, eps=1e-6)
    n_.paged_write(over, k, v, weight, weight, positions, slots, over, *pools[2:], theta=1e4, eps=1e-6)
    assert torch.equal(over, apart)
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])


@pytest.mark.parametrize("dim,page", [(128, 512), (256, 256)])
def test_pages_past_four_gigabytes(env, dim, page):
    """A cache whose last pages lie past 2^32 bytes (and 2^31 values): written, attended over by both kinds of
    launches and copied as the same pages of a small one are."""
    torch, n_ = env
    announce("paged cache past 32 bits", dim)
    pages, kv_heads, heads = 4400, 8, 16
    gen = _gen(torch, dim)
    far = torch.empty((2, pages, kv_heads, page, dim), device="cuda", dtype=torch.bfloat16)  # 9.2 GB, mostly never touched
    near = torch.randn((2, 5, kv_heads, page, dim), device="cuda", generator=gen).to(torch.bfloat16)
    far[:, -5:] = near
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    tables = ints([0, 3, 1], [4, 2, -1])
    tables_far = torch.where(tables >= 0, tables + pages - 5, tables)
    weight = torch.ones(dim, device="cuda", dtype=torch.bfloat16)
    for counts, ends in (((1, 1), (3 * page - 7, page + 9)), ((200, 1), (2 * page + 90, 2 * page))):
        rows = sum(counts)
        q, k, v = (torch.randn((rows, h, dim), device="cuda", generator=gen).to(torch.bfloat16) for h in (heads, kv_heads, kv_heads))
        positions = torch.cat([torch.arange(e - c, e) for c, e in zip(counts, ends)]).int().cuda()
        owner = torch.cat([torch.full((c,), r) for r, c in enumerate(counts)]).cuda()
        starts, outs = ints(0, counts[0], rows), []
        for pool, table in ((near, tables), (far, tables_far)):
            slots = table[owner, (positions // page).long()] * page + positions % page
            turned, out = torch.empty_like(q), torch.empty_like(q)
            n_.paged_write(q, k, v, weight, weight, positions, slots, turned, pool[0], pool[1], theta=1e6, eps=1e-6)
            n_.paged_attention(turned, pool[0], pool[1], table, starts, ints(*ends), out, dim ** -0.5)
            outs.append(out)
        assert outs[0].isfinite().all() and torch.equal(*outs)
        assert torch.equal(far[:, -5:], near)
    # a shared page, part-filled: its new owner gets the last page, copied in both planes
    refs = torch.ones(pages, dtype=torch.int32, device="cuda")
    refs[pages - 3], refs[pages - 1] = 2, 0
    chunk = [ints(0, 0, 0), ints(0, 0), ints(0, 0), ints(0), ints(0), torch.zeros((2, 2), dtype=torch.int32, device="cuda")]
    n_.paged_reserve(ints([pages - 3], [pages - 3]), ints(10, 10), refs, ints(1, 0), page, *chunk, pool=far)
    assert chunk[2].tolist() == [0, 0] and chunk[5].tolist() == [[pages - 3, pages - 1], [-1, -1]]
    assert chunk[4].tolist() == [(pages - 1) * page + 10]
    assert torch.equal(far[:, -1], near[:, 2]) and torch.equal(far[:, -5:-1], near[:, :4])
