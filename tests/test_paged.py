"""The paged cache's C ABI and wrappers without a GPU: malformed calls are refused with their codes and
messages before any device is looked for, and the model that the GPU tests compare with holds its own
invariants."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from ironmule_amd import _native
from tests.paged_model import PagedModel

P = ctypes.c_void_p
AT = 1 << 20  # an address that is never read


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_native.LIB_PATH):
        from ironmule_amd import build
        build.build()
    return _native.lib()


def _refused(lib, code, want):
    assert code == want
    got, message = _native.last_error()
    assert got == want and message


CACHE = dict(tables=AT, lengths=AT, refs=AT, requests=4, columns=8, pages=64, page_size=16)
BAD_CACHES = [({"tables": 0}, 1), ({"lengths": 0}, 1), ({"refs": 0}, 1), ({"refs": AT + 4}, 1), ({"requests": 0}, 1),
              ({"requests": 1025}, 2), ({"columns": 0}, 1), ({"columns": (1 << 20) + 1}, 2), ({"pages": 0}, 1),
              ({"page_size": 8}, 2), ({"page_size": 48}, 2), ({"page_size": 2048}, 2), ({"page_size": 0}, 2),
              ({"pages": 1 << 27}, 2), ({"columns": 1 << 20, "page_size": 1024, "pages": 4}, 0)]


def _cache(**over):
    return _native.PagedCacheDesc(**{**CACHE, **over})


CHUNK = dict(starts=AT, ends=AT, status=AT, positions=AT, slots=AT, copies=AT, rows=5)


@pytest.mark.parametrize("over,code", BAD_CACHES)
def test_a_malformed_cache_is_refused(lib, over, code):
    if code == 0:  # the largest one: refused only for the null counts
        _refused(lib, lib.imq_paged_reserve(ctypes.byref(_cache(**over)), None, ctypes.byref(_native.PagedChunkDesc(**CHUNK)),
                                            None, 0, 0, None), 1)
        return
    cache = _cache(**over)
    _refused(lib, lib.imq_paged_reserve(ctypes.byref(cache), P(AT), ctypes.byref(_native.PagedChunkDesc(**CHUNK)), None, 0, 0,
                                        None), code)
    _refused(lib, lib.imq_paged_reorder(ctypes.byref(cache), P(AT), None), code)


@pytest.mark.parametrize("over,counts,pool", [
    ({"rows": -1}, AT, None), ({"rows": (1 << 20) + 1}, AT, None), ({"starts": 0}, AT, None), ({"ends": 0}, AT, None),
    ({"status": 0}, AT, None), ({"copies": 0}, AT, None), ({"positions": 0}, AT, None), ({"slots": 0}, AT, None),
    ({}, 0, None), ({}, AT, (AT, 0, 4096)), ({}, AT, (AT, 2, 24)), ({}, AT, (AT, 2, 0)), ({}, AT, (AT + 8, 2, 4096))])
def test_a_malformed_reservation_is_refused(lib, over, counts, pool):
    chunk = _native.PagedChunkDesc(**{**CHUNK, **over})
    address, planes, size = pool or (None, 0, 0)
    _refused(lib, lib.imq_paged_reserve(ctypes.byref(_cache()), P(counts), ctypes.byref(chunk), P(address), planes, size,
                                        None), 1)
    assert lib.imq_paged_reserve(None, P(AT), ctypes.byref(chunk), None, 0, 0, None) == 1
    assert lib.imq_paged_reserve(ctypes.byref(_cache()), P(AT), None, None, 0, 0, None) == 1
    assert lib.imq_paged_reorder(ctypes.byref(_cache()), None, None) == 1


WRITE = dict(q=AT, ldq=512, k=AT, ldk=256, v=AT, ldv=256, q_norm=AT, k_norm=AT, positions=AT, slots=AT, q_out=AT, ldo=512,
             k_pages=AT, v_pages=AT, rows=3, Hq=4, Hkv=2, head_dim=128, pages=9, page_size=16, theta=1e6, eps=1e-6)


@pytest.mark.parametrize("over,code", [
    ({"q": 0}, 1), ({"k": AT + 8}, 1), ({"v": 0}, 1), ({"q_norm": 0}, 1), ({"k_norm": AT + 2}, 1), ({"positions": 0}, 1),
    ({"slots": 0}, 1), ({"q_out": 0}, 1), ({"k_pages": 0}, 1), ({"v_pages": AT + 4}, 1), ({"ldq": 504}, 1),
    ({"ldk": 252}, 1), ({"ldv": 260}, 1), ({"ldo": 0}, 1), ({"rows": -1}, 1), ({"Hq": 3}, 1), ({"Hkv": 0}, 1),
    ({"Hq": 1026, "ldq": 1 << 20, "ldo": 1 << 20}, 2), ({"head_dim": 64}, 2), ({"head_dim": 96}, 2), ({"pages": 0}, 1),
    ({"page_size": 20}, 2), ({"theta": 1.0}, 1), ({"theta": float("nan")}, 1), ({"eps": -1.0}, 1),
    ({"eps": float("nan")}, 1)])
def test_a_malformed_write_is_refused(lib, over, code):
    _refused(lib, lib.imq_paged_write(*{**WRITE, **over}.values(), None), code)


ATTEND = dict(q=AT, ldq=512, k=AT, v=AT, tables=AT, starts=AT, ends=AT, out=AT, ldo=512, rows=3, requests=2, columns=4,
              pages=9, page_size=16, Hq=4, Hkv=2, head_dim=128, max_context=64, window=0, scale=0.1)


@pytest.mark.parametrize("over,code", [
    ({"q": 0}, 1), ({"k": 0}, 1), ({"v": AT + 8}, 1), ({"tables": 0}, 1), ({"starts": 0}, 1), ({"ends": 0}, 1),
    ({"out": 0}, 1), ({"ldq": 500}, 1), ({"ldo": 516}, 1), ({"rows": -2}, 1), ({"rows": (1 << 20) + 1}, 1),
    ({"requests": 0}, 1), ({"requests": 1025}, 2), ({"columns": 0}, 1), ({"pages": 0}, 1), ({"page_size": 12}, 2),
    ({"Hq": 5}, 1), ({"Hkv": 0}, 1), ({"head_dim": 64}, 2), ({"max_context": 0}, 1), ({"window": -1}, 1),
    ({"scale": 0.0}, 1), ({"scale": -1.0}, 1), ({"scale": float("inf")}, 1), ({"scale": float("nan")}, 1)])
def test_a_malformed_attention_is_refused(lib, over, code):
    _refused(lib, lib.imq_paged_attention(*{**ATTEND, **over}.values(), P(AT), 1 << 40, None), code)


SELECT = dict(logits=AT, ld=1000, dtype=1, scores=AT, finished=AT, eos=2, groups=2, beams=4, vocab=1000, count=8, a=AT, b=AT,
              c=AT, d=AT, workspace=AT, nbytes=1 << 30)


@pytest.mark.parametrize("over,code", [
    ({"logits": 0}, 1), ({"logits": AT + 2}, 1), ({"ld": 999}, 1), ({"dtype": 2}, 1), ({"scores": 0}, 1), ({"eos": -1}, 1),
    ({"eos": 1000}, 1), ({"groups": 0}, 1), ({"beams": 0}, 1), ({"vocab": 0}, 1), ({"count": 0}, 1), ({"count": 65}, 2),
    ({"beams": 65}, 2), ({"groups": 4097}, 2), ({"groups": 4096, "beams": 64}, 2), ({"vocab": (1 << 24) + 1}, 2),
    ({"a": 0}, 1), ({"b": 0}, 1), ({"c": 0}, 1), ({"d": 0}, 1), ({"workspace": 0}, 1), ({"workspace": AT + 8}, 1),
    ({"nbytes": 64}, 1)])
def test_a_malformed_selection_is_refused(lib, over, code):
    _refused(lib, lib.imq_beam_select(*{**SELECT, **over}.values(), None), code)


def test_the_wrappers_refuse_what_does_not_fit():
    ints = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    tables, lengths, refs, counts = ints(3, 4), ints(3), ints(8), ints(3)
    chunk = [ints(4), ints(3), ints(3), ints(5), ints(5), ints(3, 2)]
    for i in range(6):  # every output of another size
        wrong = list(chunk)
        wrong[i] = ints(7)
        with pytest.raises(ValueError):
            _native.paged_reserve(tables, lengths, refs, counts, 16, *wrong)
    for bad in (tables.long(), ints(4, 3).T, ints(3, 4, 1)):
        with pytest.raises(ValueError):
            _native.paged_reserve(bad, lengths, refs, counts, 16, *chunk)
    with pytest.raises(ValueError, match="on a GPU"):
        _native.paged_reserve(tables, lengths, refs, counts, 16, *chunk)
    with pytest.raises(ValueError, match="parents"):
        _native.paged_reorder(tables, lengths, refs, ints(2), 16)
    with pytest.raises(ValueError, match="on a GPU"):
        _native.paged_reorder(tables, lengths, refs, ints(3), 16)
    pages = bf(8, 2, 16, 128)
    q, k, norm, rows = bf(5, 4, 128), bf(5, 2, 128), bf(128), ints(5)

    def write(**over):
        a = dict(q=q, k=k, v=k, q_norm=norm, k_norm=norm, positions=rows, slots=rows, q_out=q, k_pages=pages, v_pages=pages)
        return _native.paged_write(**{**a, **over}, theta=1e6, eps=1e-6)

    for over in (dict(q=q.float()), dict(q=q[:, :, :64]), dict(q=q[:4]), dict(k=bf(5, 4, 128)), dict(v=bf(4, 2, 128)),
                 dict(q=bf(5, 4, 256)[..., ::2]), dict(q=bf(5, 8, 128)[:, ::2]), dict(q=bf(5 * 516).as_strided((5, 4, 128), (516, 128, 1))),
                 dict(q_norm=bf(64)), dict(k_norm=norm.float()), dict(positions=rows.long()), dict(slots=ints(4)),
                 dict(k_pages=bf(8, 16, 2, 128).transpose(1, 2)), dict(v_pages=bf(9, 2, 16, 128)), dict(k_pages=pages.float())):
        with pytest.raises(ValueError):
            write(**over)
    with pytest.raises(ValueError, match="on a GPU"):
        write()

    def attend(**over):
        a = dict(q=q, k_pages=pages, v_pages=pages, tables=tables, starts=ints(4), ends=lengths, out=q, scale=1.0)
        return _native.paged_attention(**{**a, **over})

    for over in (dict(out=bf(5, 4, 256)), dict(starts=ints(3)), dict(ends=ints(4)), dict(tables=ints(12)), dict(q=q[0], out=q[0])):
        with pytest.raises(ValueError):
            attend(**over)
    with pytest.raises(ValueError, match="on a GPU"):
        attend()
    logits, scores = torch.zeros((6, 50)), torch.zeros(6)
    for args in ((logits.double(), scores, 3, 2), (logits, scores, 4, 2), (logits, scores[:5], 3, 2), (logits, scores, 0, 2),
                 (torch.zeros(50, 6).T, scores, 3, 2), (logits[0], scores, 1, 1), (logits, scores.double(), 3, 2)):
        with pytest.raises(ValueError):
            _native.beam_select(*args)
    with pytest.raises(ValueError, match="on a GPU"):
        _native.beam_select(logits, scores, 3, 2)


@pytest.mark.parametrize("seed", range(6))
def test_the_model_keeps_its_references(seed):
    rng = np.random.default_rng(seed)
    m = PagedModel(6, 5, 14, 16)
    for _ in range(60):
        if rng.random() < 0.4:
            m.reorder(rng.integers(-1, 7, 6))
        else:
            made = m.reserve(rng.integers(-1, 40, 6), 70)
            m.check()
            if rng.random() < 0.8:
                m.lengths = made["ends"].copy()
        m.check()
        for r in range(6):  # what a request holds has pages of its own or shared ones
            assert (m.tables[r, :-(-m.lengths[r] // 16)] >= 0).all()


def test_paged_cache_and_decoder_refuse_before_they_reach_the_gpu():
    from ironmule_amd.decode import DecoderConfig, random_weights
    from ironmule_amd.paged import PagedCache, PagedDecoder
    cfg = DecoderConfig(hidden=256, layers=1, heads=4, kv_heads=2, head_dim=128, intermediate=512, vocab=512)
    for bad in ({"requests": 0}, {"requests": 1025}, {"capacity": 0}, {"pages": 0}, {"rows": 0}, {"page_size": 8},
                {"page_size": 48}, {"page_size": 2048}):
        with pytest.raises(ValueError):
            PagedCache(cfg, **{**dict(requests=2, capacity=64, pages=8, rows=16, device="cpu"), **bad})
    cache = PagedCache(cfg, 2, 65, 8, 16, "cpu", page_size=16)
    assert cache.capacity == 80 and cache.tables.shape == (2, 5)
    assert cache.pool.shape == (2, 8, 2, 16, 128)
    for rows in (0, 17):
        with pytest.raises(ValueError):
            cache.reserve([1, 1], rows)
    with pytest.raises(ValueError):  # tensors on the host
        cache.reserve([1, 1])
    for call in (lambda: cache.fork(0, [1]), lambda: cache.fork(2, [1]), lambda: cache.fork(0, [2]),
                 lambda: cache.fork(0, [-1]), lambda: cache.release([2]), lambda: cache.release([-1])):
        with pytest.raises(ValueError):
            call()
    weights = random_weights(cfg, "cpu")
    with pytest.raises(ValueError):
        PagedDecoder(weights, PagedCache(DecoderConfig(), 1, 16, 1, 1, "cpu"))
    small = DecoderConfig(hidden=256, layers=1, heads=4, kv_heads=2, head_dim=64, intermediate=512, vocab=512)
    with pytest.raises(ValueError):
        PagedDecoder(random_weights(small, "cpu"), PagedCache(small, 1, 16, 1, 1, "cpu"))
