"""Decoding over a paged KV cache: prompts in chunks, decode steps, mixed batches, shared prefixes and
beam search, for the 4-bit decoders of this package (`decode.DecoderWeights`, `gemma3.Gemma3Weights`).

`PagedCache` holds the keys and values of several requests in pages of one pool; which page holds what
is decided on the GPU (include/ironmule_paged.h), so no step waits for the host:

    reserve   imq_paged_reserve: pages, row numbers and places of the next tokens of every request
    reorder   imq_paged_reorder: requests forked (their pages shared), reordered or ended

`PagedDecoder.extend` takes the next tokens of any number of requests, many of one and one of another,
through the model (the composition of ironmule/dense_plan.py:337-363 and
ironmule/paired_research.py:177-215):

    h = embed(tokens)                          imq_embed
    per layer:
        x = rms_norm(h)                        imq_add_rmsnorm
        q, k, v = x @ W.T                      imq_qmv_grouped up to 32 rows, else imq_prompt_matmul
        q, k = rope(norm(q)), rope(norm(k))    imq_paged_write: k and v into their pages
        o = attention(q, pages)                imq_paged_attention
        ...
    logits = rms_norm(h) @ E.T                 of the last new token of each request

`PagedDecoder.beam_search` adds imq_beam_select and reorders the beams' tables by its parents.
"""

from __future__ import annotations

import math

import torch

from . import _native
from .gemma3 import NORMS, Gemma3Weights, gelu_tanh


class PagedCache:
    """Keys and values of up to `requests` requests of at most `capacity` tokens each, in `pages` pages of
    page_size tokens, for the layers and heads of `config`; `rows`: the most new tokens of one step.

    pool (2 * layers, pages, kv_heads, page_size, head_dim) bf16: layer i's keys are pool[2 * i], its
    values pool[2 * i + 1].  tables, lengths, refs, and what a reservation gives (starts, ends, status,
    positions, slots, copies), are int32 tensors as include/ironmule_paged.h has them.  Work on a cache
    belongs on one stream at a time, the current one of its GPU."""

    def __init__(self, config, requests: int, capacity: int, pages: int, rows: int, device,
                 page_size: int = 64) -> None:
        if not 1 <= requests <= _native.MAX_PAGED_REQUESTS:
            raise ValueError(f"requests must be 1..{_native.MAX_PAGED_REQUESTS}")
        if page_size not in (16, 32, 64, 128, 256, 512, 1024):
            raise ValueError("page_size must be a power of two, 16..1024")
        if capacity < 1 or pages < 1 or rows < 1:
            raise ValueError("capacity, pages and rows must be positive")
        self.config, self.requests, self.pages, self.rows, self.page_size = config, requests, pages, rows, page_size
        columns = -(-capacity // page_size)
        self.capacity = columns * page_size

        def ints(*shape, value=0):
            return torch.full(shape, value, dtype=torch.int32, device=device)

        self.pool = torch.zeros((2 * config.layers, pages, config.kv_heads, page_size, config.head_dim),
                                dtype=torch.bfloat16, device=device)
        self.tables, self.lengths, self.refs = ints(requests, columns, value=-1), ints(requests), ints(pages)
        self.counts, self.starts, self.ends, self.status = ints(requests), ints(requests + 1), ints(requests), ints(requests)
        self.positions, self.slots = ints(rows, value=-1), ints(rows, value=-1)
        self.copies = ints(requests, 2, value=-1)

    def reserve(self, counts, rows: int | None = None) -> None:
        """Pages and rows for the next counts[r] tokens of request r (numbers, or an int32 tensor on the
        GPU); the step has `rows` rows (default: all).  `status` says which requests were refused."""
        rows = self.rows if rows is None else rows
        if not 1 <= rows <= self.rows:
            raise ValueError(f"a step of this cache has 1 to {self.rows} rows, got {rows}")
        counts = torch.as_tensor(counts, dtype=torch.int32)
        if counts.shape != (self.requests,):
            raise ValueError(f"one count for each of {self.requests} requests, got counts of shape {tuple(counts.shape)}")
        self.counts.copy_(counts)
        _native.paged_reserve(self.tables, self.lengths, self.refs, self.counts, self.page_size, self.starts,
                              self.ends, self.status, self.positions[:rows], self.slots[:rows], self.copies,
                              pool=self.pool)

    def advance(self) -> None:
        """Accepts the reserved tokens: the lengths become `ends`."""
        self.lengths.copy_(self.ends)

    def reorder(self, parents) -> None:
        """Request r becomes a copy of request parents[r] (numbers, or an int32 tensor on the GPU), sharing
        its pages; -1 ends it."""
        parents = torch.as_tensor(parents, dtype=torch.int32, device=self.tables.device)
        _native.paged_reorder(self.tables, self.lengths, self.refs, parents, self.page_size)

    def release(self, requests=None) -> None:
        """Ends these requests (default: all): their pages are free, or left to who shares them."""
        self._reparent(range(self.requests) if requests is None else requests, -1)

    def fork(self, source: int, targets) -> None:
        """The requests `targets` become copies of request `source`."""
        if not 0 <= source < self.requests:
            raise ValueError(f"request {source} is not one of {self.requests}")
        self._reparent(targets, source)

    def _reparent(self, requests, parent: int) -> None:
        parents = list(range(self.requests))
        for r in requests:
            if not 0 <= r < self.requests:
                raise ValueError(f"request {r} is not one of {self.requests}")
            parents[r] = parent
        self.reorder(parents)


class PagedDecoder:
    """A decoder over the requests of a PagedCache.  `extend` and the cache's calls launch kernels on the
    current stream and wait for nothing, so with counts and tokens on the GPU they can be captured in a HIP
    graph; the workspace of the split products belongs to this object, whose steps must not overlap."""

    def __init__(self, weights, cache: PagedCache) -> None:
        c = weights.config
        if cache.config != c:
            raise ValueError("the cache was made for another configuration")
        if c.head_dim not in (128, 256) or c.hidden > 8192:
            raise ValueError("the paged kernels take heads of 128 or 256 values, hidden sizes up to 8192")
        self.weights, self.cache, self.gemma = weights, cache, isinstance(weights, Gemma3Weights)
        self.norms = []  # Gemma's norms multiply by 1 + w, rounded to bf16
        if self.gemma:
            self.norms = [{name: 1.0 + layer[name] for name in (*NORMS, "q_norm", "k_norm")} for layer in weights.layers]
            self.final_norm = 1.0 + weights.norm
        shapes = [*c.projections.values(), (c.vocab, c.hidden)]
        device = weights.norm.device
        self.workspace = torch.zeros(_native.qmv_workspace_bytes(shapes) // 4 + 1, dtype=torch.float32, device=device)

    def _project(self, names, x: torch.Tensor, weights, dtype=torch.bfloat16) -> list[torch.Tensor]:
        """x @ W.T for 4-bit weights of one layer: one sweep of each weight up to 32 rows, else the products
        for many rows."""
        quants = [weights[name] for name in names]
        if x.shape[0] > _native.MAX_ROWS:
            return [_native.prompt_matmul(*quant, x, out_dtype=dtype) for quant in quants]
        return _native.qmv_grouped(quants, [x] * len(quants), out_dtype=dtype, workspace=self.workspace)

    def _tokens(self, tokens: torch.Tensor, rows: int) -> torch.Tensor:
        """The token of each row: rows are those of the requests that were taken, in order."""
        starts = self.cache.starts
        row = torch.arange(rows, dtype=torch.int32, device=tokens.device)
        owner = torch.searchsorted(starts[1:], row, right=True, out_int32=True)
        used, owner = owner < self.cache.requests, owner.clamp_(max=self.cache.requests - 1)
        place = (row - starts[owner]).clamp_(0, tokens.shape[1] - 1)
        return torch.where(used, tokens[owner, place], 0)

    def _attend(self, i: int, layer, q, k, v, q_norm, k_norm, theta, scale, window, max_context) -> torch.Tensor:
        c, cache, rows = self.weights.config, self.cache, q.shape[0]
        k_pages, v_pages = cache.pool[2 * i], cache.pool[2 * i + 1]
        q = q.view(rows, c.heads, c.head_dim)
        _native.paged_write(q, k.view(rows, c.kv_heads, c.head_dim), v.view(rows, c.kv_heads, c.head_dim), q_norm, k_norm,
                            cache.positions[:rows], cache.slots[:rows], q, k_pages, v_pages, theta, c.eps)
        out = torch.empty_like(q)
        _native.paged_attention(q, k_pages, v_pages, cache.tables, cache.starts, cache.ends, out, scale, window=window,
                                max_context=max_context)
        return out.view(rows, c.heads * c.head_dim)

    def extend(self, tokens, counts, rows: int | None = None, max_context: int | None = None) -> torch.Tensor:
        """Takes the next counts[r] tokens of every request r, tokens[r][0 .. counts[r] - 1], through the
        model and into the cache; returns the fp32 logits (requests, vocab) of the last one of each.  A
        request without new tokens, or one the cache refused (cache.status: no pages, no rows), has NaN
        logits and is left as it was.

        tokens: lists of numbers per request, or an int32 tensor (requests, width) on the GPU with counts
        there too; then `rows` bounds the sum of the counts (default: the cache's rows, or requests *
        width if that is less), and a request with a count past its tokens is refused (status 2).  max_context
        bounds the requests' lengths and only plans the launches (default: what the cache's tables can hold;
        short contexts in a large cache are faster with their own bound).  A token outside the vocabulary makes
        its request's logits NaN from then on."""
        c, cache = self.weights.config, self.cache
        device, limits = cache.pool.device, None
        if not isinstance(tokens, torch.Tensor):
            if len(tokens) != cache.requests:
                raise ValueError(f"one list of tokens for each of {cache.requests} requests")
            if not isinstance(counts, torch.Tensor) and any(n > len(t) for n, t in zip(counts, tokens)):
                raise ValueError("a count is more than its request's tokens")
            limits = [len(t) for t in tokens]
            width = max(1, *limits)
            tokens = torch.tensor([list(t) + [0] * (width - len(t)) for t in tokens], dtype=torch.int32).to(device)
        if tokens.dtype != torch.int32 or tokens.dim() != 2 or tokens.shape[0] != cache.requests or tokens.shape[1] < 1:
            raise ValueError(f"tokens must be int32 ({cache.requests}, width)")
        if tokens.device != device:
            raise ValueError(f"the tokens are on {tokens.device}, the cache on {device}")
        if not isinstance(counts, torch.Tensor):
            if len(counts) != cache.requests or min(counts) < 0 or max(counts) > tokens.shape[1]:
                raise ValueError(f"{cache.requests} counts of 0 to {tokens.shape[1]} tokens, got {counts}")
            total = sum(counts)
            if total > cache.rows:
                raise ValueError(f"a step of this cache has at most {cache.rows} rows, got {total}")
            rows = max(1, total) if rows is None else rows
        else:  # (-1: malformed, which the reservation refuses)
            limit = tokens.shape[1] if limits is None else torch.tensor(limits, dtype=torch.int32).to(counts.device)
            counts = counts.masked_fill(counts > limit, -1)
        if rows is None:
            rows = min(cache.rows, cache.requests * tokens.shape[1])
        cache.reserve(counts, rows)
        h = torch.empty((rows, c.hidden), dtype=torch.float32, device=device)
        _native.embed(*self.weights.embed, self._tokens(tokens, rows), h)
        h, delta = (self._gemma_layers if self.gemma else self._layers)(h, max_context)
        last = (cache.starts[1:] - 1).clamp_(min=0)
        h = h.index_select(0, last)
        x = torch.empty(h.shape, dtype=torch.bfloat16, device=device)
        if self.gemma:
            _native.add_rmsnorm(h, self.final_norm, x, c.eps)
        else:
            _native.add_rmsnorm(h, self.weights.norm, x, c.eps, delta=None if delta is None else delta.index_select(0, last))
        logits, = self._project(["embed"], x, {"embed": self.weights.embed}, torch.float32)
        logits.masked_fill_((cache.starts[1:] == cache.starts[:-1])[:, None], float("nan"))
        cache.advance()
        return logits

    def _layers(self, h: torch.Tensor, max_context):
        c, rows = self.weights.config, h.shape[0]
        x = torch.empty(h.shape, dtype=torch.bfloat16, device=h.device)
        delta = None
        for i, layer in enumerate(self.weights.layers):
            _native.add_rmsnorm(h, layer["input_norm"], x, c.eps, delta=delta)
            q, k, v = self._project(("q", "k", "v"), x, layer)
            o = self._attend(i, layer, q, k, v, layer["q_norm"], layer["k_norm"], c.theta, c.head_dim ** -0.5, 0, max_context)
            delta, = self._project(("o",), o, layer)
            _native.add_rmsnorm(h, layer["post_norm"], x, c.eps, delta=delta)
            act = torch.empty((rows, c.intermediate), dtype=torch.bfloat16, device=h.device)
            if 5 <= rows <= _native.MAX_ROWS and c.hidden % 256 == 0:
                _native.gate_up_silu(layer["gate"], layer["up"], x, act)
            else:
                _native.silu_mul(*self._project(("gate", "up"), x, layer), act)
            delta, = self._project(("down",), act, layer)
        return h, delta

    def _gemma_layers(self, h: torch.Tensor, max_context):
        """The residual stream holds bf16 values (each sum rounded), in fp32 for the norms."""
        c = self.weights.config
        scale = float(torch.tensor(math.sqrt(c.hidden), dtype=torch.bfloat16))
        h = (h.to(torch.bfloat16).float() * scale).to(torch.bfloat16).float()

        def norm(rows, weight):
            return _native.add_rmsnorm(rows, weight, torch.empty(rows.shape, dtype=torch.bfloat16, device=h.device), c.eps)

        for i, (layer, norms) in enumerate(zip(self.weights.layers, self.norms)):
            theta, window = (c.theta_global, 0) if c.is_global(i) else (c.theta_local, c.window)
            q, k, v = self._project(("q", "k", "v"), norm(h, norms["input_norm"]), layer)
            o = self._attend(i, layer, q, k, v, norms["q_norm"], norms["k_norm"], theta, c.query_scalar ** -0.5, window,
                             max_context)
            o, = self._project(("o",), o, layer)
            h = (h + norm(o.float(), norms["post_attn_norm"])).to(torch.bfloat16).float()
            gate, up = self._project(("gate", "up"), norm(h, norms["pre_ff_norm"]), layer)
            act = (gelu_tanh(gate.float()).to(torch.bfloat16).float() * up.float()).to(torch.bfloat16)
            down, = self._project(("down",), act, layer)
            h = (h + norm(down.float(), norms["post_ff_norm"])).to(torch.bfloat16).float()
        return h, None

    def prefill(self, prompts) -> torch.Tensor:
        """Appends prompts[r] (a list of tokens, may be empty) to every request r, in chunks of at most the
        cache's rows; returns the logits (requests, vocab) of the last token of each (NaN where it is
        empty).  Raises RuntimeError if the cache has not the pages: a request then holds the chunks of its prompt
        up to the first that did not fit, as many tokens more as its length says."""
        cache = self.cache
        if len(prompts) != cache.requests:
            raise ValueError(f"one prompt for each of {cache.requests} requests")
        prompts = [list(p) for p in prompts]
        at, logits = [0] * cache.requests, None
        refused = torch.zeros_like(cache.status)
        while logits is None or any(a < len(p) for a, p in zip(at, prompts)):
            room, counts = cache.rows, []
            for a, p in zip(at, prompts):
                counts.append(min(room, len(p) - a))
                room -= counts[-1]
            chunks = [p[a:a + n] for a, p, n in zip(at, prompts, counts)]
            if logits is None:
                logits = self.extend(chunks, counts)
            else:  # (nothing more of a request that was refused a chunk)
                new = torch.tensor(counts, dtype=torch.int32).to(logits.device)
                chunk = self.extend(chunks, torch.where(refused == 0, new, 0), rows=max(1, sum(counts)))
                logits = torch.where((new > 0)[:, None], chunk, logits)
            refused |= cache.status
            at = [a + n for a, n in zip(at, counts)]
        if bool(refused.any()):
            raise RuntimeError("the cache has too few pages, or a request too few columns, for these prompts")
        return logits

    def beam_search(self, prompts, beams: int, steps: int, eos: int = -1):
        """The `beams` continuations of up to `steps` tokens that beam search finds for each prompt: (tokens
        int32 (prompts, beams, steps), scores fp32 (prompts, beams): the sums of their log probabilities,
        the best first).  A continuation ends with token `eos` (-1: none does), which fills what is left of
        it (every step is launched all the same, as nothing waits for the tokens); where there are fewer than
        `beams` continuations the tokens are -1, the score -inf.  The cache has len(prompts) * beams requests, which are ended first; the beams' requests are left in it, without
        their last tokens.  Raises RuntimeError if the cache has not the pages."""
        cache, groups = self.cache, len(prompts)
        if groups < 1 or beams < 1 or groups * beams != cache.requests:
            raise ValueError(f"{groups} prompts of {beams} beams do not fill {cache.requests} requests")
        if steps < 1 or any(len(p) < 1 for p in prompts):
            raise ValueError("a search needs a step, and prompts of at least one token")
        device = cache.pool.device
        cache.release()
        first = [[] for _ in range(cache.requests)]
        for g, prompt in enumerate(prompts):
            first[g * beams] = prompt
        logits = self.prefill(first)  # the other beams' are NaN: they offer nothing
        scores = torch.zeros(cache.requests, dtype=torch.float32, device=device)
        finished = None if eos < 0 else torch.zeros(cache.requests, dtype=torch.int32, device=device)
        history = torch.empty((cache.requests, steps), dtype=torch.int32, device=device)
        refused = torch.zeros_like(cache.status)
        for step in range(steps):
            scores, parents, chosen, ended = (
                t.reshape(-1) for t in _native.beam_select(logits, scores, beams, beams, finished=finished, eos=eos))
            finished = None if eos < 0 else ended
            history = history.index_select(0, parents.clamp(min=0))
            history[:, step] = chosen
            history.masked_fill_((parents < 0)[:, None], -1)
            cache.reorder(parents)
            if step + 1 < steps:
                going = (parents >= 0) & (ended == 0)
                logits = self.extend(chosen.clamp(min=0)[:, None], going.int(), rows=min(cache.requests, cache.rows))
                refused |= cache.status
        if bool(refused.any()):
            raise RuntimeError("the cache has too few pages, columns or rows for this search")
        return history.view(groups, beams, steps), scores.view(groups, beams)
