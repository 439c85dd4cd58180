"""Greedy generation over paged KV caches: sequences join, grow and leave on their own.

Where Batch32Generator decodes a fixed batch in lock-step over contiguous caches,
a PagedGenerator keeps a pool of pages per layer.  A sequence is added with any
prompt, may be extended later (a chat turn), and is released when done; every
step() runs one forward pass over whatever is pending: one token of each decoding
sequence, and chunks of the prompts that are still being read.
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

    def _plan(self) -> list[tuple[int, int]]:
        """(sequence, tokens of it) of the next step, within chunk_tokens and the free pages."""
        ready = [(i, s) for i, s in self.sequences.items() if s.pending]
        ready.sort(key=lambda x: len(x[1].pending) > 1)  # single tokens first, else in order
        room, pages, plan = self.chunk_tokens, len(self.free_pages), []
        for i, s in ready:
            n = min(len(s.pending), room)
            have = len(s.pages) * self.page_size - s.length
            n = min(n, have + pages * self.page_size, self.max_seq_len - s.length)
            if n > 0:
                pages -= max(0, -(-(n - have) // self.page_size))
                room -= n
                plan.append((i, n))
        return plan

    # ---- steps -----------------------------------------------------------------
    def step(self, keep_logits: bool = False) -> dict[int, int]:
        """One forward pass over pending tokens.  Returns the next token of every
        sequence whose pending tokens are all read; it becomes that sequence's next
        pending token."""
        plan = self._plan()
        if not plan:
            if any(s.pending for s in self.sequences.values()):
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
        """Greedy continuation of prompts of any lengths: max_new_tokens tokens each."""
        if max_new_tokens < 1:
            raise ValueError("max_new_tokens must be positive")
        if any(len(np.asarray(p).reshape(-1)) + max_new_tokens - 1 > self.max_seq_len for p in prompts):
            raise ValueError("prompt + max_new_tokens exceeds max_seq_len")
        todo = [self.add(p) for p in prompts]
        out: dict[int, list[int]] = {}
        try:
            while len(out) < len(todo):
                self.step()
                for i in todo:
                    if i in self.sequences and len(self.sequences[i].generated) >= max_new_tokens:
                        out[i] = self.sequences[i].generated[:max_new_tokens]
                        self.release(i)
        finally:
            for i in todo:
                if i in self.sequences:
                    self.release(i)
        return [out[i] for i in todo]
