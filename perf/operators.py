"""Serving over a paged cache, timed operator by operator: cases, their inputs, one pass of each in
plain torch operations or through the framework's kernels, and what each pass computes in 64 bits.

Kinds of case:

    round    a scheduler's round on the tables of a paged cache: requests that have ended give their
             pages back, beams are forked from their prompt (`paged_reorder`), then every request's new
             tokens get pages, rows and slots, and the part-filled pages that forks share are copied
             (`paged_reserve`)
    write    per-head norm and rotary of q and k, and k and v into the pages (`paged_write`)
    attend   attention of the requests' new tokens over their pages: a token each, chunks of prompts
             over what is cached already, or both in one batch (`paged_attention`)
    select   the best continuations of beams over the whole vocabulary (`beam_select`)

A cache is `tables` (requests, columns) of page numbers, -1 where there is none, `lengths`, and `refs`,
how many table entries hold each page; the pages of one layer's keys or values are (pages, kv_heads,
page size, head size).  A page is held by several requests only after a fork, in the same column of each.
"""

import math
import random
from types import SimpleNamespace

import torch

own = False
DEVICE = "cuda"
EPS, THETA = 1e-6, 1e6


def listed():
    return [
        # a beam search step of one prompt: eight beams forked again from a prompt of 1000 tokens
        dict(name="round_beams_8", kind="round", running=0, entering=0, forks=8, context=1000, prompt=1, page=16,
             pages=2048, kv_heads=8, head_dim=128, mix=1),
        # a serving batch: 48 running requests, 16 that leave to new prompts, two sets of four beams
        dict(name="round_serving_72", kind="round", running=48, entering=16, forks=8, context=4096, prompt=700, page=16,
             pages=16384, kv_heads=8, head_dim=128, mix=2),
        # a full node's round: 500 running requests and 200 prompts entering a cache of 131072 pages
        dict(name="round_node_764", kind="round", running=500, entering=200, forks=64, context=2500, prompt=2500, page=16,
             pages=131072, kv_heads=1, head_dim=128, mix=3),
        # one layer's q, k and v of a small decode batch
        dict(name="write_step_5", kind="write", rows=5, heads=32, kv_heads=8, head_dim=128, page=16, positions=9000, mix=4),
        # one layer's q, k and v of a batch of prompt chunks with padding rows, heads of 256
        dict(name="write_chunk_4099", kind="write", rows=4099, heads=16, kv_heads=8, head_dim=256, page=64,
             positions=30000, mix=5),
        # one conversation, a token at a time
        dict(name="attend_step_1x777", kind="attend", form="step", requests=1, tokens=1, context=777, heads=32, kv_heads=8,
             head_dim=128, page=16, window=0, mix=6),
        # a serving batch's step over long and short conversations
        dict(name="attend_step_32x8000", kind="attend", form="step", requests=32, tokens=1, context=8000, heads=32,
             kv_heads=8, head_dim=128, page=16, window=0, mix=7),
        # the last chunk of a long prompt
        dict(name="attend_chunk_1024_of_16384", kind="attend", form="chunk", requests=1, tokens=1024, context=16384, heads=32,
             kv_heads=8, head_dim=128, page=64, window=0, mix=8),
        # prompts' chunks and running requests in one batch
        dict(name="attend_mixed_24", kind="attend", form="mixed", requests=24, tokens=509, context=3001, heads=32, kv_heads=8,
             head_dim=128, page=32, window=0, mix=9),
        # a sliding-window layer with heads of 256, chunks and steps
        dict(name="attend_window_7", kind="attend", form="mixed", requests=7, tokens=700, context=6000, heads=16, kv_heads=8,
             head_dim=256, page=16, window=1024, mix=10),
        # one prompt's four beams over the vocabulary
        dict(name="select_1x4", kind="select", groups=1, beams=4, count=4, vocab=151936, bf16=False, finished=0, mix=11),
        # a batch of eight beam searches, two candidates for each beam, bf16 logits (many equal ones)
        dict(name="select_8x4_bf16", kind="select", groups=8, beams=4, count=8, vocab=262144, bf16=True, finished=3, mix=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("round", "write", "attend", "attend", "attend", "select"))
    mix = rng.randint(0, 1 << 20)
    if kind == "round":
        running, entering, forks = _log(rng, 1, 500), _log(rng, 1, 200), rng.choice((0, 4, 8, 32))
        page = rng.choice((16, 32, 64, 128))
        context, prompt = _log(rng, 20, 2500), _log(rng, 1, 2500)
        most = (running + forks + 2 * entering + 3) * (max(context, prompt) // page + 2)
        return dict(kind=kind, running=running, entering=entering, forks=forks, context=context, prompt=prompt, page=page,
                    pages=min(131072, max(64, int(most * rng.uniform(0.9, 2.0)))), kv_heads=1, head_dim=128, mix=mix)
    if kind == "write":
        heads, kv_heads, head_dim = rng.choice(((32, 8, 128), (16, 8, 128), (16, 8, 256), (5, 5, 128), (7, 1, 256)))
        return dict(kind=kind, rows=_log(rng, 1, 4099), heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    page=rng.choice((16, 32, 64, 128)), positions=_log(rng, 100, 30000), mix=mix)
    if kind == "attend":
        form = rng.choice(("step", "chunk", "mixed"))
        heads, kv_heads, head_dim = rng.choice(((32, 8, 128), (16, 8, 128), (16, 8, 256), (12, 12, 128), (20, 4, 128), (8, 1, 256)))
        requests = _log(rng, 1, 48) if form == "step" else _log(rng, 1, 24)
        tokens = 1 if form == "step" else _log(rng, 2, min(1024, 4096 // requests))
        most = 28_000_000 // (requests * kv_heads * head_dim * (1 if form == "step" else 4))
        context = max(tokens, _log(rng, 1, min(16384, most)))
        return dict(kind=kind, form=form, requests=requests, tokens=tokens, context=context, heads=heads, kv_heads=kv_heads,
                    head_dim=head_dim, page=rng.choice((16, 32, 64, 128)), window=rng.choice((0, 0, 1024, _log(rng, 1, 4000))),
                    mix=mix)
    beams = _log(rng, 1, 16)
    return dict(kind=kind, groups=_log(rng, 1, max(1, 32 // beams)), beams=beams, count=beams * rng.choice((1, 2)),
                vocab=_log(rng, 1000, 262144), bf16=rng.random() < 0.4, finished=rng.choice((0, 1, 5)), mix=mix)


# ------------------------------------------------------------------ what a case stands for

def _requests(case):
    """(new tokens, tokens cached after them) of each request of an attend case."""
    rng, made = random.Random(case["mix"]), []
    for i in range(case["requests"]):
        n = 1
        if case["form"] == "chunk" or (case["form"] == "mixed" and i % 4 == 0):
            n = case["tokens"] if i == 0 else _log(rng, 1, case["tokens"])
        if i and rng.random() < 0.05:
            n = 0  # a request that waits
        length = case["context"] if i == 0 else rng.randint(max(1, case["context"] // 4), case["context"])
        made.append((n, max(n, length)))
    return made


def _round(case):
    """(length, new tokens, parent) of each request of a round: running ones, ones that leave to a new
    prompt, and forks of the first; request 0 is the prompt that the beams are forked from."""
    rng, made = random.Random(case["mix"]), []
    for i in range(1 + case["running"] if case["forks"] else max(1, case["running"])):
        made.append((case["context"] if i == 0 else rng.randint(1, case["context"]), 1 if i or not case["forks"] else 0, i))
    for _ in range(case["entering"]):
        made.append((rng.randint(1, case["context"]), rng.randint(max(1, case["prompt"] // 4), case["prompt"]), -1))
    for _ in range(case["forks"]):
        made.append((0, 1, 0))
    return made


def _columns(case):
    return max(case["context"], case["prompt"]) // case["page"] + 2


# ------------------------------------------------------------------ inputs

def _generator(seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    return gen


def _normal(gen, *shape):
    return torch.randn(shape, device=DEVICE, generator=gen).to(torch.bfloat16)


def _norm_weight(gen, n):
    return torch.empty(n, device=DEVICE).uniform_(0.9, 1.1, generator=gen).to(torch.bfloat16)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _tables(gen, needs, columns, pages):
    """Tables whose row r holds needs[r] pages, scattered over the cache as after some time of serving."""
    order = torch.randperm(pages, device=DEVICE, generator=gen).to(torch.int32)
    need = _ints(needs)
    rank = need.cumsum(0) - need
    column = torch.arange(columns, device=DEVICE)
    held = column[None] < need[:, None]
    at = (rank[:, None] + column[None]).clamp(max=pages - 1)
    return torch.where(held, order[at], -1).contiguous()


def prepare(case, seed):
    gen, kind = _generator(seed), case["kind"]
    s = SimpleNamespace(kind=kind, case=case)
    if kind == "round":
        made, page = _round(case), case["page"]
        pages, columns, count = case["pages"], _columns(case), len(made)
        needs, left = [], pages
        for length, _, _ in made:
            needs.append(min(-(-length // page), left))
            left -= needs[-1]
        s.tables = _tables(gen, needs, columns, pages)
        s.lengths = _ints([min(length, need * page) for (length, _, _), need in zip(made, needs)])
        s.refs = torch.zeros(pages, dtype=torch.int32, device=DEVICE)
        s.refs.index_add_(0, s.tables.clamp(min=0).flatten(), (s.tables >= 0).int().flatten())
        s.counts, s.parents = _ints([c for _, c, _ in made]), _ints([p for _, _, p in made])
        s.pool = _normal(gen, 2, pages, case["kv_heads"], page, case["head_dim"])
        s.rows, s.page = sum(c for _, c, _ in made), page
        empty = torch.full((3 * count + 1 + 2 * s.rows + 2 * count,), -1, dtype=torch.int32, device=DEVICE)
        s.starts, s.ends, s.status, s.positions, s.slots, s.copies = empty.split(
            (count + 1, count, count, s.rows, s.rows, 2 * count))
        s.copies = s.copies.view(count, 2)
        return s
    if kind == "write":
        rows, d, page = case["rows"], case["head_dim"], case["page"]
        pages = rows // page + 3
        s.q, s.k, s.v = (_normal(gen, rows, h, d) for h in (case["heads"], case["kv_heads"], case["kv_heads"]))
        s.q_norm, s.k_norm = _norm_weight(gen, d), _norm_weight(gen, d)
        s.positions = torch.randint(0, case["positions"], (rows,), device=DEVICE, generator=gen).to(torch.int32)
        s.slots = torch.randperm(pages * page, device=DEVICE, generator=gen)[:rows].to(torch.int32)
        if rows > 16:  # a batch padded to its size
            s.slots[-3:] = -1
        s.q_out = torch.zeros((rows, case["heads"], d), dtype=torch.bfloat16, device=DEVICE)
        s.k_pages = torch.zeros((pages, case["kv_heads"], page, d), dtype=torch.bfloat16, device=DEVICE)
        s.v_pages = torch.zeros_like(s.k_pages)
        return s
    if kind == "attend":
        made, page, d = _requests(case), case["page"], case["head_dim"]
        needs = [-(-length // page) for _, length in made]
        pages = sum(needs) + 5
        s.tables = _tables(gen, needs, max(needs) + 1, pages)
        s.k_pages = _normal(gen, pages, case["kv_heads"], page, d)
        s.v_pages = _normal(gen, pages, case["kv_heads"], page, d)
        counts = [n for n, _ in made]
        s.rows, s.most, s.context = sum(counts), max(counts), max(length for _, length in made)
        s.starts = _ints([sum(counts[:i]) for i in range(len(counts) + 1)])
        s.ends = _ints([length for _, length in made])
        s.q = _normal(gen, s.rows, case["heads"], d)
        s.out = torch.empty_like(s.q)
        s.scale = d ** -0.5
        return s
    rows = case["groups"] * case["beams"]
    logits = 3.0 * torch.randn((rows, case["vocab"]), device=DEVICE, generator=gen)
    s.logits = logits.to(torch.bfloat16) if case["bf16"] else logits
    s.scores = -12.0 * torch.rand(rows, device=DEVICE, generator=gen)
    s.finished = torch.zeros(rows, dtype=torch.int32, device=DEVICE)
    if case["finished"]:
        s.finished[torch.randperm(rows, device=DEVICE, generator=gen)[:min(rows // 2, case["finished"])]] = 1
    return s


# ------------------------------------------------------------------ the plain forms

def _index(n):
    return torch.arange(n, device=DEVICE)


def _plain_reorder(s):
    count, columns = s.tables.shape
    row, parent = _index(count), s.parents.long()
    keep = (parent == row) | (parent < -1) | (parent >= count)
    source = parent.clamp(0, count - 1)
    length = torch.where(parent < 0, 0, s.lengths[source])
    held = (_index(columns)[None] * s.page < length[:, None])
    new = torch.where(held, s.tables[source], -1)
    new = torch.where(keep[:, None], s.tables, new)
    for table, sign in ((s.tables, -1), (new, 1)):
        s.refs.index_add_(0, table.clamp(min=0).flatten(), (sign * (table >= 0)).int().flatten())
    s.tables.copy_(new)
    s.lengths.copy_(torch.where(keep, s.lengths, length))


def _plain_reserve(s):
    count, columns = s.tables.shape
    pages, page = s.refs.shape[0], s.page
    column = _index(columns)
    length, new, tables = s.lengths.long(), s.counts.long(), s.tables.long()
    bad = (new < 0) | (length < 0) | (length + new > columns * page)
    new = torch.where(bad, 0, new)
    first, end = length // page, length + new
    current = tables.gather(1, first.clamp(0, columns - 1)[:, None])[:, 0]
    shared = (new > 0) & (current >= 0) & (s.refs[current.clamp(min=0)] > 1)
    written = (column[None] >= first[:, None]) & (column[None] * page < end[:, None]) & (new > 0)[:, None]
    need = written & ((tables < 0) | (shared[:, None] & (column[None] == first[:, None])))
    wants = need.sum(1)
    free = (s.refs == 0).sum()
    short = (wants > 0) & (wants.cumsum(0) > free)
    full = (new > 0) & (new.cumsum(0) > s.rows)
    take = ~bad & ~short & ~full
    order = torch.argsort((s.refs != 0).int(), stable=True)  # the free pages, lowest first
    rank = need.flatten().long().cumsum(0) - 1
    given = torch.where(need & take[:, None], order[rank.clamp(0, pages - 1)].view(count, columns), -1)
    leave = shared & take
    s.refs.index_add_(0, current.clamp(min=0), -leave.int())
    s.refs.index_add_(0, given.clamp(min=0).flatten(), (given >= 0).int().flatten())
    tables = torch.where(given >= 0, given, tables)
    taken = torch.where(take, new, 0)
    s.tables.copy_(tables)
    s.starts[0] = 0
    s.starts[1:].copy_(taken.cumsum(0))
    s.ends.copy_(length + taken)
    s.status.copy_(torch.where(bad, 2, torch.where(short, 1, torch.where(full, 3, 0))))
    at = _index(s.rows)
    of = torch.searchsorted(s.starts[1:].contiguous().long(), at, right=True).clamp(max=count - 1)
    position = length[of] + at - s.starts[:-1].long()[of]
    slot = tables[of, (position // page).clamp(0, columns - 1)] * page + position % page
    live = at < s.starts[-1]
    s.positions.copy_(torch.where(live, position, -1))
    s.slots.copy_(torch.where(live, slot, -1))
    copied = leave & (length % page > 0)
    target = tables.gather(1, first.clamp(0, columns - 1)[:, None])[:, 0]
    s.copies.copy_(torch.where(copied[:, None], torch.stack([current, target], 1), -1))
    s.pool[:, target[copied]] = s.pool[:, current[copied]]


def _plain_write(s):
    d = s.case["head_dim"]
    frequency = THETA ** (-torch.arange(d // 2, dtype=torch.float64, device=DEVICE) * 2.0 / d)
    angle = s.positions.double()[:, None] * frequency
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(x, weight):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
        lo, hi = x[..., :d // 2], x[..., d // 2:]
        return torch.cat([lo * cos - hi * sin, lo * sin + hi * cos], -1).to(torch.bfloat16)

    live = s.slots >= 0
    s.q_out.copy_(torch.where(live[:, None, None], turn(s.q, s.q_norm), s.q_out))
    page, offset = (s.slots[live].long() // s.case["page"]), (s.slots[live].long() % s.case["page"])
    s.k_pages[page, :, offset] = turn(s.k, s.k_norm)[live]
    s.v_pages[page, :, offset] = s.v[live]


def _plain_attend(s):
    c = s.case
    count, d, page = c["requests"], c["head_dim"], c["page"]
    group = c["heads"] // c["kv_heads"]
    columns = -(-s.context // page)
    held = s.tables[:, :columns].clamp(min=0).long()

    def keys(pages):  # (requests, kv heads, context, head size)
        return pages[held].float().transpose(1, 2).reshape(count, c["kv_heads"], columns * page, d)

    n = (s.starts[1:] - s.starts[:-1]).long()
    new = _index(s.most)
    row = (s.starts[:-1].long()[:, None] + new[None]).clamp(max=s.rows - 1)
    q = s.q[row].float().view(count, s.most, c["kv_heads"], group, d).permute(0, 2, 1, 3, 4)
    q = q.reshape(count, c["kv_heads"], s.most * group, d)
    position = (s.ends.long() - n)[:, None] + new[None]
    at = _index(columns * page)
    seen = at[None, None] <= position[..., None]
    if c["window"]:
        seen &= at[None, None] > position[..., None] - c["window"]
    seen &= (new[None] < n[:, None])[..., None] & (at[None] < s.ends[:, None])[:, None]
    seen = seen.repeat_interleave(group, 1)[:, None]
    scores = torch.matmul(q, keys(s.k_pages).transpose(2, 3).contiguous()).mul_(s.scale).masked_fill_(~seen, float("-inf"))
    scores = scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = scores.sum(-1, keepdim=True)
    # (a page row past a request's end may hold anything: it is not multiplied)
    values = torch.where((at[None] < s.ends[:, None])[:, None, :, None], keys(s.v_pages), 0.0)
    out = torch.matmul(scores, values) / total
    out = out.view(count, c["kv_heads"], s.most, group, d).permute(0, 2, 1, 3, 4).reshape(count, s.most, c["heads"], d)
    s.out.copy_(out[new[None] < n[:, None]].to(torch.bfloat16))


EOS = 2


def _plain_select(s):
    c = s.case
    x, score = s.logits.double(), s.scores.double()
    most = x.amax(-1, keepdim=True)
    key = score[:, None] + ((x - most) - (x - most).exp().sum(-1, keepdim=True).log())
    done = s.finished.bool()[:, None]
    token = _index(c["vocab"])[None]
    key = torch.where(done, torch.where(token == EOS, score[:, None], float("-inf")), key)
    best, at = torch.sort(key.view(c["groups"], -1), dim=-1, descending=True, stable=True)
    best, at = best[:, :c["count"]], at[:, :c["count"]]
    parent = at // c["vocab"] + c["beams"] * _index(c["groups"])[:, None]
    token, dead = at % c["vocab"], best == float("-inf")
    ended = torch.where(dead, 0, (s.finished.long()[parent] | (token == EOS)).int())
    return (best.float(), torch.where(dead, -1, parent).int(), torch.where(dead, -1, token).int(), ended.int())


# ------------------------------------------------------------------ one pass

def run(s):
    if own:
        from ironmule_amd import _native as n
    if s.kind == "round":
        if own:
            n.paged_reorder(s.tables, s.lengths, s.refs, s.parents, s.page)
            n.paged_reserve(s.tables, s.lengths, s.refs, s.counts, s.page, s.starts, s.ends, s.status, s.positions, s.slots,
                            s.copies, pool=s.pool)
        else:
            _plain_reorder(s)
            _plain_reserve(s)
        return dict(tables=s.tables, lengths=s.lengths, refs=s.refs, starts=s.starts, ends=s.ends, status=s.status,
                    positions=s.positions, slots=s.slots, copies=s.copies, pool=s.pool)
    if s.kind == "write":
        if own:
            n.paged_write(s.q, s.k, s.v, s.q_norm, s.k_norm, s.positions, s.slots, s.q_out, s.k_pages, s.v_pages, THETA, EPS)
        else:
            _plain_write(s)
        return s.q_out, s.k_pages, s.v_pages
    if s.kind == "attend":
        if own:
            return n.paged_attention(s.q, s.k_pages, s.v_pages, s.tables, s.starts, s.ends, s.out, s.scale,
                                     window=s.case["window"])
        _plain_attend(s)
        return s.out
    if own:
        return n.beam_select(s.logits, s.scores, s.case["beams"], s.case["count"], finished=s.finished, eos=EOS)
    return _plain_select(s)


# ------------------------------------------------------------------ what a pass cannot do without

def _pairs(n, length, window):
    """(query, key) pairs that n new tokens at the end of `length` see, and the keys that any of them sees."""
    first = length - n
    if not window:
        return n * first + n * (n + 1) // 2, length if n else 0
    pairs = sum(min(first + i + 1, window) for i in range(n))
    return pairs, min(length, n + window - 1) if n else 0


def work(case):
    kind = case["kind"]
    if kind == "round":
        made, page = _round(case), case["page"]
        entries, given, copied = 0, 0, 0
        for i, (length, new, parent) in enumerate(made):
            fork = parent >= 0 and parent != i
            length = made[parent][0] if fork else 0 if parent < 0 else length
            entries += -(-length // page)
            given += -(-(length + new) // page) - -(-length // page)
            copied += 1 if fork and length % page else 0
        rows = sum(new for _, new, _ in made)
        plane = 2 * case["kv_heads"] * page * case["head_dim"] * 2
        # the held entries read, the changed ones and their references written, maps, copies
        return dict(bytes=4 * (entries + 4 * given + 9 * len(made) + 2 * rows) + 2 * copied * plane, flops=0)
    d = case.get("head_dim")
    if kind == "write":
        live = case["rows"] - (3 if case["rows"] > 16 else 0)
        heads = case["heads"] + 2 * case["kv_heads"]
        return dict(bytes=live * (4 * heads * d + 8) + 4 * d, flops=live * (case["heads"] + case["kv_heads"]) * d * 7)
    if kind == "attend":
        pairs = [_pairs(n, length, case["window"]) for n, length in _requests(case)]
        rows = sum(n for n, _ in _requests(case))
        return dict(bytes=4 * d * (rows * case["heads"] + sum(k for _, k in pairs) * case["kv_heads"]),
                    flops=4 * d * case["heads"] * sum(p for p, _ in pairs))
    rows = case["groups"] * case["beams"]
    live = rows - min(rows // 2, case["finished"])
    return dict(bytes=live * case["vocab"] * (2 if case["bf16"] else 4) + rows * 8 + case["groups"] * case["count"] * 16,
                flops=3 * live * case["vocab"])


# ------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "round":
        return None
    if kind == "write":
        return _exact_write(s)
    return _exact_attend(s) if kind == "attend" else _exact_select(s)


def _exact_write(s):
    d, page = s.case["head_dim"], s.case["page"]
    pair = torch.arange(0, d, 2, device=DEVICE, dtype=torch.float64) / d
    turn = s.positions.double()[:, None, None] * torch.exp(-math.log(THETA) * pair)
    turn = torch.complex(turn.cos(), turn.sin())

    def head(x, weight):
        x = x.double()
        x = x / (x.square().sum(-1, keepdim=True) / d + EPS).sqrt() * weight.double()
        z = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:].contiguous()) * turn
        return torch.cat([z.real, z.imag], -1)

    q, k, v = s.q_out.double(), s.k_pages.double(), s.v_pages.double()
    live = (s.slots >= 0).nonzero()[:, 0]
    slot = s.slots[live].long()
    q[live] = head(s.q, s.q_norm)[live]
    k[slot // page, :, slot % page] = head(s.k, s.k_norm)[live]
    v[slot // page, :, slot % page] = s.v[live].double()
    return q, k, v


def _exact_attend(s):
    c, out = s.case, torch.zeros(s.q.shape, dtype=torch.float64, device=DEVICE)
    group, page, row = c["heads"] // c["kv_heads"], c["page"], 0
    for r, (n, length) in enumerate(_requests(c)):
        if not n:
            continue
        held = s.tables[r, :-(-length // page)].long()
        k, v = (p[held].permute(1, 0, 2, 3).flatten(1, 2)[:, :length].double() for p in (s.k_pages, s.v_pages))
        position = torch.arange(length - n, length, device=DEVICE)[:, None]
        at = torch.arange(length, device=DEVICE)[None]
        hidden = (at > position) | ((at <= position - c["window"]) if c["window"] else False)
        for head in range(c["heads"]):
            q = s.q[row:row + n, head].double()
            p = ((q @ k[head // group].T) * s.scale).masked_fill(hidden, float("-inf")).softmax(-1)
            out[row:row + n, head] = p @ v[head // group]
        row += n
    return out


def _exact_select(s):
    c = s.case
    key = torch.log_softmax(s.logits.double(), -1) + s.scores.double()[:, None]
    for row in s.finished.nonzero()[:, 0].tolist():
        key[row] = float("-inf")
        key[row, EOS] = s.scores[row].double()
    best = key.view(c["groups"], -1).topk(c["count"], dim=-1).values
    return best, None, None, None
