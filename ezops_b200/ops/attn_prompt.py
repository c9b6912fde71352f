"""Causal grouped-query attention of a step's tokens over paged KV caches.

``AttnDecodeOp`` (ezops/ops/attn_decode.py:9-67) has one query per row; here row b brings n_b = cu_tokens[b+1] -
cu_tokens[b] of them - a prompt, a piece of a prompt behind a cached context, a single token, or none - whose keys and
values are already in the pools as the last n_b of its ``seq_lens[b]`` keys.  Query i of the row sees the keys
0 .. seq_lens[b] - n_b + i::

    out = softmax(q K^T / sqrt(D)) V           (a query that sees no key gives zeros)

Q, out [T, H, D] bf16 (rows of one step behind each other, token rows may lie further apart); K_pool, V_pool [pages,
NKV, page_size, D]; page_table [batch, max_pages], seq_lens [batch], cu_tokens [batch + 1] int32 - the tensors of a
``PagedPlan``.  Rows of ``out`` behind ``cu_tokens[batch]`` are left as they were; T may be 0.  What the pools hold behind a row's last key
is never used.  Equal calls give equal bits; the order of a row's sums may depend on the other rows.
"""

from __future__ import annotations

import torch

from ..registry import get_kernel
from .base_op import Op


class AttnPromptOp(Op):
    _params_desc = {
        "batch": "Rows (requests)",
        "tokens": "Tokens of the step that gen_data makes (calls take any number)",
        "num_heads": "Number of query heads",
        "head_dim": "Dimension per head (64 or 128)",
        "max_pages": "Page table entries per row",
        "page_size": "Keys per page (a power of two >= 64)",
        "num_kv_heads": "Number of KV heads for GQA (default: num_heads)",
    }
    _atol = 1e-2
    _rtol = 1e-2

    def __init__(self, batch: int, tokens: int, num_heads: int, head_dim: int, max_pages: int, page_size: int, backend: str = "ref",
                 num_kv_heads: int | None = None):
        self.batch, self.tokens, self.num_heads, self.head_dim = batch, tokens, num_heads, head_dim
        self.max_pages, self.page_size = max_pages, page_size
        self.num_kv_heads = num_heads if num_kv_heads is None else num_kv_heads
        if min(batch, tokens, num_heads, self.num_kv_heads, max_pages) < 1:
            raise ValueError("batch, tokens, num_heads, num_kv_heads and max_pages must be positive")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim ({head_dim}) must be 64 or 128")
        if num_heads % self.num_kv_heads != 0:
            raise ValueError(f"num_heads ({num_heads}) must be divisible by num_kv_heads ({self.num_kv_heads})")
        if num_heads // self.num_kv_heads > 128:
            raise ValueError("at most 128 query heads per kv head")
        if page_size < 64 or page_size & (page_size - 1):
            raise ValueError(f"page_size ({page_size}) must be a power of two >= 64")
        self._backend = backend
        if backend == "ref":
            self._kernel = self._ref_forward
        else:
            self._kernel = get_kernel("attn_prompt", backend)(batch, num_heads, head_dim, max_pages, page_size,
                                                              num_kv_heads=self.num_kv_heads)

    def forward(self, Q, K_pool, V_pool, page_table, seq_lens, cu_tokens, out=None):
        return self._kernel(Q, K_pool, V_pool, page_table, seq_lens, cu_tokens, out)

    def gen_data(self, device="cuda"):
        """Tokens dealt out evenly, contexts of different lengths in front of them."""
        B, T, page, P = self.batch, self.tokens, self.page_size, self.max_pages
        cu = torch.arange(B + 1) * T // B
        new = cu.diff()
        lens = torch.minimum(new + torch.randint(0, P * page, (B,)), torch.tensor(P * page))
        used = (lens + page - 1) // page
        pages = int(used.sum()) + 1
        table = torch.full((B, P), -1, dtype=torch.int64)
        table[torch.arange(P) < used[:, None]] = torch.randperm(pages)[: pages - 1]
        kw = dict(device=device, dtype=torch.bfloat16)
        Q = torch.randn(T, self.num_heads, self.head_dim, **kw)
        K_pool, V_pool = (torch.randn(pages, self.num_kv_heads, page, self.head_dim, **kw) for _ in range(2))
        return Q, K_pool, V_pool, *(t.to(torch.int32).to(device) for t in (table, lens, cu))

    def _ref_forward(self, Q, K_pool, V_pool, page_table, seq_lens, cu_tokens, out=None):
        NKV, D, page = self.num_kv_heads, self.head_dim, self.page_size
        out = torch.empty_like(Q) if out is None else out
        cu, lens = cu_tokens.tolist(), seq_lens.tolist()
        for b, n in enumerate(lens):
            m = cu[b + 1] - cu[b]
            if m == 0:
                continue
            pages = page_table[b, : -(-n // page)].long()
            k, v = (t[pages].float().transpose(0, 1).reshape(NKV, -1, D)[:, :n] for t in (K_pool, V_pool))
            q = Q[cu[b] : cu[b + 1]].float().view(m, NKV, -1, D).permute(1, 2, 0, 3)  # [NKV, G, m, D]
            seen = torch.arange(n, device=Q.device) <= n - m + torch.arange(m, device=Q.device)[:, None]
            s = (q @ k[:, None].transpose(-1, -2) * D**-0.5).masked_fill(~seen, float("-inf"))
            p = torch.softmax(s, dim=-1).masked_fill(~seen, 0.0)  # rows without a key are NaN before
            out[cu[b] : cu[b + 1]] = (p @ v[:, None]).permute(2, 0, 1, 3).reshape(m, -1, D).to(out.dtype)
        return out
