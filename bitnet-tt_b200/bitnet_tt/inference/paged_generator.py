"""Greedy generation over paged KV caches: sequences join, grow and leave on their own.

Where Batch32Generator decodes a fixed batch in lock-step over contiguous caches,
a PagedGenerator keeps a pool of pages per layer.  A sequence is added with any
prompt, may be extended later (a chat turn), and is released when done; every
step() runs one forward pass over whatever is pending: one token of each decoding
sequence, and chunks of the prompts that are still being read.  Prompts take pages
in the order they were added, and only what decoding sequences and the prompts
before them leave, so that one that has been begun can be read to its end.
"""

from __future__ import annotations

from dataclasses import dataclass, field
from typing import Sequence

import numpy as np
import torch

from ..layers.paged_kv import PagedBatch
from ..utils.rope import half_split_tables


@dataclass
class _Sequence:
    pages: list[int] = field(default_factory=list)
    length: int = 0                                   # tokens in the cache
    pending: list[int] = field(default_factory=list)  # tokens still to be read
    generated: list[int] = field(default_factory=list)
    limit: int | None = None                          # the length it will end at, if that is known


class PagedGenerator:
    def __init__(self, model, num_pages: int, page_size: int = 64, cache_dtype: torch.dtype = torch.bfloat16,
                 max_seq_len: int | None = None, chunk_tokens: int = 8192) -> None:
        """num_pages pages of page_size tokens in each layer's pool.  chunk_tokens
        bounds the tokens of one step (and its activations): decoding sequences
        come first, prompts share the rest in the order they were added."""
        cfg = model.config
        if num_pages < 1 or chunk_tokens < 1:
            raise ValueError("num_pages and chunk_tokens must be positive")
        self.model = model
        self.device = model.device
        self.page_size = page_size
        self.max_seq_len = max_seq_len or cfg.max_position_embeddings
        self.chunk_tokens = chunk_tokens
        self.caches = model.paged_caches(num_pages, page_size, cache_dtype)
        cos, sin = half_split_tables(cfg.head_dim, self.max_seq_len, cfg.rope_theta)
        self.rope = (cos.to(self.device), sin.to(self.device))
        self.free_pages = list(range(num_pages - 1, -1, -1))
        self.sequences: dict[int, _Sequence] = {}
        self._next_id = 0
        self.last_logits: torch.Tensor | None = None  # of the last step, when it was asked for them

    # ---- sequences -----------------------------------------------------------
    def _tokens(self, tokens: Sequence[int]) -> list[int]:
        out = [int(t) for t in np.asarray(tokens).reshape(-1)]
        if not out:
            raise ValueError("at least one token is needed")
        if min(out) < 0 or max(out) >= self.model.config.vocab_size:
            raise ValueError("token id out of range")
        return out

    def add(self, prompt: Sequence[int]) -> int:
        """A new sequence; its prompt is read by the next steps."""
        tokens = self._tokens(prompt)
        if len(tokens) > self.max_seq_len:
            raise ValueError("prompt longer than max_seq_len")
        self._next_id += 1
        self.sequences[self._next_id] = _Sequence(pending=tokens)
        return self._next_id

    def extend(self, seq: int, tokens: Sequence[int]) -> None:
        """Appends tokens (a user's next turn) behind what the sequence holds."""
        s = self.sequences[seq]
        more = self._tokens(tokens)
        if s.length + len(s.pending) + len(more) > self.max_seq_len:
            raise ValueError("sequence longer than max_seq_len")
        s.pending += more

    def release(self, seq: int) -> None:
        """Ends a sequence and gives its pages back."""
        self.free_pages += self.sequences.pop(seq).pages

    def _more_pages(self, s: _Sequence, length: int) -> int:
        """Pages that it needs beyond its own to hold `length` tokens."""
        return max(0, -(-length // self.page_size) - len(s.pages))

    def _plan(self, only: set[int] | None) -> list[tuple[int, int]]:
        """(sequence, tokens of it) of the next step, within chunk_tokens and the free pages."""
        ready = [(i, s) for i, s in self.sequences.items() if s.pending and (only is None or i in only)]
        ready.sort(key=lambda x: len(x[1].pending) > 1)  # single tokens first, else in order
        room, pages, plan, late = self.chunk_tokens, len(self.free_pages), [], []

        def take(i: int, s: _Sequence, pages: int) -> int:
            """Plans what fits; the pages that it costs."""
            nonlocal room
            n = min(len(s.pending), room, len(s.pages) * self.page_size - s.length + pages * self.page_size,
                    self.max_seq_len - s.length)
            if n <= 0:
                return 0
            room -= n
            plan.append((i, n))
            return self._more_pages(s, s.length + n)

        # What the decoding sequences need next: all of it where their end is known, else a page each.
        kept = 0
        for i, s in ready:
            if len(s.pending) == 1:
                used = take(i, s, pages)
                pages -= used
                more = self._more_pages(s, s.limit if s.limit is not None else self.max_seq_len) - used
                kept += max(0, more) if s.limit is not None else min(1, max(0, more))
        for i, s in ready:
            if len(s.pending) == 1:
                continue
            end = max(s.length + len(s.pending), s.limit or 0)
            rest = self._more_pages(s, min(end, self.max_seq_len))
            if rest > pages - kept:
                late.append((i, s))  # it cannot be read to its end: not while anything else goes on
                continue
            take(i, s, pages)
            pages -= rest  # whatever is not taken now is kept for it
        if not plan:
            for i, s in late:
                pages -= take(i, s, pages)
        return plan

    # ---- steps -----------------------------------------------------------------
    def step(self, keep_logits: bool = False) -> dict[int, int]:
        """One forward pass over pending tokens.  Returns the next token of every
        sequence whose pending tokens are all read; it becomes that sequence's next
        pending token.  RuntimeError when nothing that is pending fits the free pages
        (release a sequence, then go on)."""
        return self._step(None, keep_logits)

    def _step(self, only: set[int] | None, keep_logits: bool = False) -> dict[int, int]:
        plan = self._plan(only)
        if not plan:
            if any(s.pending for i, s in self.sequences.items() if only is None or i in only):
                raise RuntimeError("no pages or positions left for the pending tokens")
            return {}
        ids, pages, lens = [], [], []
        for i, n in plan:
            s = self.sequences[i]
            while len(s.pages) * self.page_size < s.length + n:
                s.pages.append(self.free_pages.pop())
            ids += s.pending[:n]
            pages.append(s.pages)
            lens.append(s.length + n)
        batch = PagedBatch.of([n for _, n in plan], lens, pages, self.device)
        with torch.cuda.device(self.device):
            nxt, self.last_logits = self.model.forward_paged(torch.tensor(ids, dtype=torch.int32, device=self.device), batch,
                                                             self.rope, self.caches, keep_logits)
        tokens, out = nxt.tolist(), {}
        for (i, n), t in zip(plan, tokens):
            s = self.sequences[i]
            s.length += n
            del s.pending[:n]
            if not s.pending:
                s.generated.append(t)
                out[i] = t
                if s.length < self.max_seq_len:
                    s.pending.append(t)
        return out

    def generate(self, prompts: Sequence[Sequence[int]], max_new_tokens: int = 128) -> list[list[int]]:
        """Greedy continuation of prompts of any lengths: max_new_tokens tokens each.
        Prompts start as the pages for all of their tokens are there, in order; a
        batch may be larger than the pool.  Other sequences stay as they are."""
        if max_new_tokens < 1:
            raise ValueError("max_new_tokens must be positive")
        todo = [self._tokens(p) for p in prompts]
        lengths = [len(p) + max_new_tokens - 1 for p in todo]
        if any(n > self.max_seq_len for n in lengths):
            raise ValueError("prompt + max_new_tokens exceeds max_seq_len")
        need = [-(-n // self.page_size) for n in lengths]
        room = len(self.free_pages)  # nothing but what this call starts takes any until it ends
        if any(n > room for n in need):
            raise ValueError(f"prompt + max_new_tokens needs more than the {room} free pages")
        out: list[list[int]] = [[] for _ in todo]
        active: dict[int, int] = {}  # sequence -> prompt
        at = 0
        try:
            while at < len(todo) or active:
                while at < len(todo) and need[at] <= room:
                    seq = self.add(todo[at])
                    self.sequences[seq].limit = lengths[at]
                    active[seq] = at
                    room -= need[at]
                    at += 1
                self._step(set(active))
                for seq in list(active):
                    if len(self.sequences[seq].generated) >= max_new_tokens:
                        i = active.pop(seq)
                        out[i] = self.sequences[seq].generated[:max_new_tokens]
                        room += need[i]
                        self.release(seq)
        finally:
            for seq in active:
                self.release(seq)
        return out
