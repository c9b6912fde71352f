"""The plan of a step over paged KV caches, made on the GPU from the requests' lengths.

A serving step takes ``new_lens[b]`` new tokens of request b (a prompt, a piece of one, a single token, or none) behind
its ``ctx_lens[b]`` cached ones.  Before the model runs, the pages that the new tokens need are taken from a free list and
entered into the page table, and every token gets its position and its cache slot::

    held(n) = ceil(n / page_size)
    page_table[b, held(ctx) : held(ctx + new)] = the next pages from the end of free_pages[:free_count], row by row
    seq_lens = ctx_lens + new_lens        cu_tokens = running sum of new_lens, from 0
    token t of row b:  position = ctx_lens[b] + t - cu_tokens[b]
                       slot = page_table[b, position // page_size] * page_size + position % page_size

``positions`` has one axis and counts the tokens of a row; a program with positions of its own (images: several axes, and text
behind them that does not go on at its place in the cache) takes the slots and offsets from here and brings its positions.

All tensors are int32.  ``page_table`` [batch, max_pages] is changed in place; the other results come in a ``PagedPlan``
whose tensors have fixed sizes, so that a step can be captured in a CUDA graph: ``positions`` and ``slots`` hold -1 behind
the last token, and tokens beyond ``max_tokens`` are dropped.  ``free_count`` [1] counts what is left; it is negative when the
list was too short, and the table entries and slots of the missing pages are -1.  A row holds ``max_pages * page_size`` positions:
tokens beyond them keep their place in the step with slot -1, and ``seq_lens`` stops there.  Such a row has to be ended before its
step: ``seq_lens`` no longer counts all of its tokens, from which attention tells what each of them sees.  The reference has
contiguous caches only (ezops/ops/attn_decode.py:52-56).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from ..registry import get_kernel
from .base_op import Op


class PagedPlan(NamedTuple):
    seq_lens: torch.Tensor  # [batch]
    cu_tokens: torch.Tensor  # [batch + 1]
    positions: torch.Tensor  # [max_tokens]
    slots: torch.Tensor  # [max_tokens]
    free_count: torch.Tensor  # [1]


class PagedPlanOp(Op):
    _params_desc = {
        "batch": "Rows (requests) of the page table",
        "max_tokens": "Tokens that a step can hold",
        "max_pages": "Page table entries per row",
        "page_size": "Keys per page (a power of two >= 64)",
        "num_pages": "Pages in each pool",
    }

    def __init__(self, batch: int, max_tokens: int, max_pages: int, page_size: int, num_pages: int, backend: str = "ref"):
        for name, value in (("batch", batch), ("max_tokens", max_tokens), ("max_pages", max_pages), ("num_pages", num_pages)):
            if value < 1:
                raise ValueError(f"{name} ({value}) must be positive")
        if page_size < 64 or page_size & (page_size - 1):
            raise ValueError(f"page_size ({page_size}) must be a power of two >= 64")
        self.batch, self.max_tokens, self.max_pages = batch, max_tokens, max_pages
        self.page_size, self.num_pages = page_size, num_pages
        self._backend = backend
        if backend == "ref":
            self._kernel = self._ref_forward
        else:
            self._kernel = get_kernel("paged_plan", backend)(batch, max_tokens, max_pages, page_size, num_pages)

    def new_plan(self, device="cuda") -> PagedPlan:
        """Tensors for ``out=``: a serving loop keeps one plan and has every step written into it."""
        sizes = (self.batch, self.batch + 1, self.max_tokens, self.max_tokens, 1)
        return PagedPlan(*(torch.empty(n, dtype=torch.int32, device=device) for n in sizes))

    def forward(self, ctx_lens, new_lens, page_table, free_pages, free_count, out: PagedPlan | None = None) -> PagedPlan:
        if out is None:
            out = self.new_plan(ctx_lens.device)
        self._kernel(ctx_lens, new_lens, page_table, free_pages, free_count, out)
        return out

    def check(self, actual, expected) -> bool:
        return all(torch.equal(a, e) for a, e in zip(actual, expected))

    def gen_data(self, device="cuda"):
        """A batch whose cached contexts use about half of the pools, single tokens next to a few prompts."""
        B, P, page = self.batch, self.max_pages, self.page_size
        most = min(P, max(1, self.num_pages // (2 * B)))  # pages a row may hold
        ctx = torch.randint(0, most * page + 1, (B,))
        new = torch.ones(B, dtype=torch.int64)
        for b in range(0, B, 4):
            new[b] = 1 + torch.randint(0, max(1, min(self.max_tokens // B, page)), (1,)).item()
        new = torch.minimum(new, P * page - ctx)
        held = (ctx + page - 1) // page
        order = torch.randperm(self.num_pages)
        table = torch.full((B, P), -1, dtype=torch.int64)
        n = int(held.sum())
        table[torch.arange(P) < held[:, None]] = order[:n]
        free = torch.cat([order[n:], torch.full((n,), -1)])
        return tuple(t.to(torch.int32).to(device) for t in (ctx, new, table, free, torch.tensor([self.num_pages - n])))

    def _ref_forward(self, ctx_lens, new_lens, page_table, free_pages, free_count, out: PagedPlan) -> None:
        page, T = self.page_size, self.max_tokens
        cap, free = self.max_pages * page, free_pages.tolist()
        left = min(int(free_count), len(free))
        lens, cu, positions, slots = [], [0], [], []
        valid = lambda i: i if 0 <= i < self.num_pages else -1  # noqa: E731
        for b in range(self.batch):
            ctx = min(max(int(ctx_lens[b]), 0), cap)
            n = min(max(int(new_lens[b]), 0), T - cu[-1])
            lens.append(min(ctx + n, cap))
            cu.append(cu[-1] + n)
            for j in range(-(-ctx // page), -(-lens[-1] // page)):
                left -= 1
                page_table[b, j] = valid(free[left]) if left >= 0 else -1
            for pos in range(ctx, ctx + n):
                positions.append(pos)
                at = valid(int(page_table[b, pos // page])) if pos < cap else -1
                slots.append(at * page + pos % page if at >= 0 else -1)
        pad = [-1] * (T - len(slots))
        for dst, src in zip(out, (lens, cu, positions + pad, slots + pad, [left])):
            dst.copy_(torch.tensor(src, dtype=torch.int32))
