"""Reservations whose every number is written down from the words of include/ironmule_paged.h: which
requests are refused, why, and which pages the others get."""

from __future__ import annotations

import pytest

from tests.conftest import gpu_available
from tests.gpu_util import announce

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]

PAGE = 16


def _reserve(tables, lengths, refs, counts, rows):
    """(tables, refs, starts, ends, status, slots, copies) after a reservation, as lists."""
    import torch

    from ironmule_amd import _native
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    n = len(lengths)
    tables, refs = ints(tables), ints(refs)
    made = [torch.full(s, -7, dtype=torch.int32, device="cuda") for s in ((n + 1,), (n,), (n,), (rows,), (rows,), (n, 2))]
    _native.paged_reserve(tables, ints(lengths), refs, ints(counts), PAGE, *made)
    starts, ends, status, positions, slots, copies = (t.tolist() for t in made)
    assert all((p < 0) == (s < 0) and (s < 0 or s % PAGE == p % PAGE) for p, s in zip(positions, slots))
    return dict(tables=tables.tolist(), refs=refs.tolist(), starts=starts, ends=ends, status=status, slots=slots, copies=copies)


@pytest.mark.parametrize("pages,rows,status", [
    (6, 100, [0, 2, 2, 0, 0]), (5, 100, [0, 2, 2, 0, 1]), (4, 100, [0, 2, 2, 1, 1]), (6, 60, [0, 2, 2, 0, 3]),
    (6, 59, [0, 2, 2, 3, 3]), (5, 60, [0, 2, 2, 0, 1]), (1, 100, [1, 2, 2, 1, 1]), (6, 0, [3, 2, 2, 3, 3])])
def test_each_reason_to_refuse(pages, rows, status):
    """20, -1, 70 (of 64 that its columns hold), 40 and 1 new tokens: pages and rows run out where the sums of the
    well-formed ones do, a refused one's among them; a request without pages is said to lack those first."""
    announce("paged refusals", pages, rows)
    got = _reserve([[-1] * 4 for _ in range(5)], [0] * 5, [0] * pages, [20, -1, 70, 40, 1], rows)
    assert got["status"] == status
    counts = [n if s == 0 else 0 for n, s in zip([20, -1, 70, 40, 1], status)]
    assert got["ends"] == counts and got["starts"] == [sum(counts[:i]) for i in range(6)]
    given = {0: [0, 1], 3: [2, 3, 4], 4: [5]}
    for r in range(5):
        want = given.get(r, []) if status[r] == 0 else []
        assert got["tables"][r] == want + [-1] * (4 - len(want))
    assert got["refs"] == [int(any(p in given.get(r, []) and status[r] == 0 for r in range(5))) for p in range(pages)]
    assert got["slots"] == [given[r][i // PAGE] * PAGE + i % PAGE for r in range(5) for i in range(counts[r])] + [-1] * (
        rows - sum(counts))
    assert got["copies"] == [[-1, -1]] * 5


@pytest.mark.parametrize("pages,rows,status", [(8, 100, [2, 0, 0]), (6, 100, [2, 0, 1]), (8, 52, [2, 0, 3]), (8, 32, [2, 3, 3])])
def test_a_shared_page_past_the_tokens_counts_as_asked_for(pages, rows, status):
    """Request 0 gave tokens up past whole pages that request 1 holds too: refused, but the page that it would
    have had instead of its first, shared one, and its 30 rows, are counted."""
    announce("paged refusals, shared past the tokens", pages, rows)
    got = _reserve([[0, 1, 2, -1], [0, 1, 2, -1], [-1] * 4], [10, 48, 0], [2, 2, 2] + [0] * (pages - 3), [30, 3, 20], rows)
    assert got["status"] == status
    assert got["ends"] == [10, 48 + 3 * (status[1] == 0), 20 * (status[2] == 0)]
    assert got["tables"] == [[0, 1, 2, -1], [0, 1, 2, 4 if status[1] == 0 else -1],
                             [5, 6, -1, -1] if status[2] == 0 else [-1] * 4]
    taken = {4: status[1] == 0, 5: status[2] == 0, 6: status[2] == 0}
    assert got["refs"] == [2, 2, 2] + [int(taken.get(p, False)) for p in range(3, pages)]
