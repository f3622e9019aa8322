"""A paged cache's tables in plain Python, request by request, and attention in 64 bits: what the paged
tests compare the kernels with."""

from __future__ import annotations

import numpy as np


class PagedModel:
    """Tables, lengths and references as lists; `reserve` and `reorder` follow the C header's words."""

    def __init__(self, requests: int, columns: int, pages: int, page_size: int) -> None:
        self.tables = np.full((requests, columns), -1, np.int32)
        self.lengths = np.zeros(requests, np.int32)
        self.refs = np.zeros(pages, np.int32)
        self.page = page_size

    def reserve(self, counts, rows: int):
        requests, columns = self.tables.shape
        free = [int(p) for p in np.flatnonzero(self.refs == 0)]
        starts, ends, status = [0], [], []
        copies = np.full((requests, 2), -1, np.int32)
        positions, slots = np.full(rows, -1, np.int32), np.full(rows, -1, np.int32)
        asked_pages = asked_rows = 0
        refs = self.refs.copy()  # as they were at the call: what is shared
        for r in range(requests):
            length, new = int(self.lengths[r]), int(counts[r])
            bad = length < 0 or new < 0 or length + new > columns * self.page
            new = 0 if bad else new
            first = length // self.page
            need = []
            for c in range(first, (length + new - 1) // self.page + 1 if new else first):
                page = int(self.tables[r, c])
                held = 0 <= page < len(refs)
                if held and refs[page] > 1 and c > first:
                    bad = True
                if not held or (c == first and refs[page] > 1):
                    need.append(c)
            ranks = range(asked_pages, asked_pages + len(need))
            asked_pages += len(need)
            asked_rows += new
            state = 2 if bad else 1 if need and asked_pages > len(free) else 3 if new and asked_rows > rows else 0
            status.append(state)
            new = 0 if state else new
            if state == 0:
                for c, k in zip(need, ranks):
                    old, page = int(self.tables[r, c]), free[k]
                    if 0 <= old < len(refs):
                        self.refs[old] -= 1
                        if length % self.page:
                            copies[r] = old, page
                    self.tables[r, c] = page
                    self.refs[page] = 1
            for i in range(new):
                position = length + i
                positions[starts[-1] + i] = position
                slots[starts[-1] + i] = self.tables[r, position // self.page] * self.page + position % self.page
            starts.append(starts[-1] + new)
            ends.append(length + new)
        return dict(starts=np.array(starts, np.int32), ends=np.array(ends, np.int32), status=np.array(status, np.int32),
                    positions=positions, slots=slots, copies=copies)

    def reorder(self, parents) -> None:
        tables, lengths = self.tables.copy(), self.lengths.copy()
        requests, columns = tables.shape
        for r, p in enumerate(int(v) for v in parents):
            if p == r or not -1 <= p < requests:
                continue
            for c in range(columns):
                held = p >= 0 and lengths[p] > c * self.page
                page = int(tables[p, c]) if held else -1
                for old, change in ((int(tables[r, c]), -1), (page, 1)):
                    if 0 <= old < len(self.refs):
                        self.refs[old] += change
                self.tables[r, c] = page
            self.lengths[r] = lengths[p] if p >= 0 else 0

    def check(self) -> None:
        """What has to hold of any cache: references count the entries."""
        held = self.tables[self.tables >= 0]
        assert np.array_equal(np.bincount(held, minlength=len(self.refs)), self.refs)


def attention(torch, q, k_pages, v_pages, tables, starts, ends, scale, window=0):
    """(out, bound) in float64 of every row that a request has (others NaN): the definition, and how far
    a kernel may be off that rounds probabilities to bf16 and keeps the rest in fp32.  With u = 2^-24, a score of D
    terms is off by at most (D + 8) u S, S the row's largest scale sum |q k|, and moves its probability's share by
    that much relatively, twice (numerator and sum); a sum over L keys in blocks of 16 or more adds (L / 16 + 64) u
    twice; rounding a probability to bf16 2^-8 of it; all of them of A = sum p |v|.  The output's rounding: 2^-8."""
    rows, heads, dim = q.shape
    pages, kv_heads, page, _ = k_pages.shape
    group, u = heads // kv_heads, 2.0 ** -24
    out = torch.full((rows, heads, dim), float("nan"), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    starts, ends = starts.tolist(), ends.tolist()
    for r, end in enumerate(ends):
        n = starts[r + 1] - starts[r]
        if n < 1:
            continue
        held = tables[r, :-(-end // page)].long()
        good = ((held >= 0) & (held < pages)).repeat_interleave(page)[:end]
        held = torch.where((held >= 0) & (held < pages), held, 0)
        k, v = (t[held].permute(1, 0, 2, 3).flatten(1, 2)[:, :end].double() for t in (k_pages, v_pages))
        at, position = (torch.arange(m, device=q.device) for m in (end, n))
        position = position + end - n
        seen = (at[None] <= position[:, None]) & good[None]
        if window:
            seen &= at[None] > position[:, None] - window
        for h in range(heads):
            x = q[starts[r]:starts[r + 1], h].double()
            kh, vh = k[h // group], v[h // group]
            s = (x @ kh.T) * scale
            large = torch.where(seen, (x.abs() @ kh.abs().T) * scale, 0.0).amax(-1, keepdim=True)
            s = torch.where(seen, s, float("-inf"))
            p = torch.where(seen, (s - s.amax(-1, keepdim=True)).exp(), 0.0)
            # a key that no row sees may hold anything; one that only some see must not reach the others
            some = torch.where(seen.any(0)[:, None], vh, 0.0)
            clean = torch.where(some.isfinite(), some, 0.0)
            total = p.sum(-1, keepdim=True)
            o = (p @ clean) / total
            for j in (~some.isfinite()).any(-1).nonzero()[:, 0].tolist():
                add = p[:, j:j + 1] / total * torch.where(some[j].isfinite(), 0.0, some[j])[None]
                o = o + torch.where(seen[:, j:j + 1], add, 0.0)
            o = torch.where(seen.any(-1, keepdim=True), o, 0.0)
            a = torch.where(seen.any(-1, keepdim=True), (p @ clean.abs()) / total, 0.0)
            out[starts[r]:starts[r + 1], h] = o
            relative = 2.0 ** -8 + 2 * (dim + 8) * u * large + 2 * (end / 16 + 64) * u
            bound[starts[r]:starts[r + 1], h] = 2.0 ** -8 * o.abs() + relative * a + 1e-30
    return out, bound
