"""Per-head QK RMSNorm, rotary embedding and the write into paged KV caches for the tokens of a step.

What ``FusedQkNormRopeOp`` (ezops/ops/fused_qk_norm_rope.py:7-169) does for one token per row into contiguous caches,
here for any number of tokens, straight from the rows of the fused projection and into page pools::

    q, k, v = qkv[:, :H*D], qkv[:, H*D:(H+NKV)*D], qkv[:, (H+NKV)*D:]
    q_out = rope(rmsnorm(q) * q_norm_w)
    K_pool[slot // page_size, :, slot % page_size] = rope(rmsnorm(k) * k_norm_w) ;  V_pool[...] = v

Norm through rotation stay in fp32 with a single rounding to bf16; the rotation is the rotate_half form against tables
[max_positions, head_dim] whose second half repeats the first.

Images and video have positions of several axes (time, height, width): ``positions`` is [axes, T] then, and frequency
i < D/2 is turned by the position of its axis.  ``sections`` holds the number of frequencies per axis (they add up to
D/2).  Chunked (default): the first ``sections[0]`` frequencies belong to axis 0, the next to axis 1, ...  ``interleaved``:
axis a > 0 has the frequencies a + axes*j for j < sections[a], axis 0 all others.  One axis is the ordinary rotation;
equal positions on all axes give its result.  Behind an image the position of a token is no longer its place in the cache:
single tokens of such a request come through this operator as well, since ``Qwen3DecodeStackOp`` rotates a token by its slot.

A token with a negative position is padding (nothing is written for it), a token with a negative slot is not cached.
Tensors (bf16 unless noted): qkv [T, (H+2*NKV)*D], rows may lie further apart; q_norm_w, k_norm_w [D] or None (unit);
cos, sin [max_positions, D]; positions int32 [T] or [axes, T]; slots int32 [T]; K_pool, V_pool [num_pages, NKV,
page_size, D].  Returns q_out [T, H, D]; T may be 0.
"""

from __future__ import annotations

import torch

from ..registry import get_kernel
from .base_op import Op


def axis_of_frequency(sections, interleaved: bool) -> list[int]:
    """The position axis of each of the D/2 frequencies."""
    axes, half = len(sections), sum(sections)
    if interleaved:
        return [i % axes if i // axes < sections[i % axes] else 0 for i in range(half)]
    return [a for a, n in enumerate(sections) for _ in range(n)]


class PagedQkNormRopeOp(Op):
    _params_desc = {
        "tokens": "Tokens of the step that gen_data makes (calls take any number)",
        "num_heads": "Number of query heads",
        "head_dim": "Dimension per head (64 or 128)",
        "max_positions": "Rows of the cos/sin tables",
        "page_size": "Keys per page (a power of two >= 64)",
        "num_pages": "Pages in each pool",
        "num_kv_heads": "Number of KV heads for GQA (default: num_heads)",
        "sections": "Frequencies per position axis, adding up to head_dim / 2 (default: one axis)",
        "interleaved": "Axes take turns along the frequencies instead of one range each",
    }
    _atol = 1e-2
    _rtol = 1e-2

    rms_eps = 1e-6
    rope_theta = 1e6

    def __init__(self, tokens: int, num_heads: int, head_dim: int, max_positions: int, page_size: int, num_pages: int,
                 backend: str = "ref", num_kv_heads: int | None = None, sections=None, interleaved: bool = False):
        self.tokens, self.num_heads, self.head_dim, self.max_positions = tokens, num_heads, head_dim, max_positions
        self.num_kv_heads = num_heads if num_kv_heads is None else num_kv_heads
        self.page_size, self.num_pages = page_size, num_pages
        if min(tokens, num_heads, self.num_kv_heads, max_positions, num_pages) < 1:
            raise ValueError("tokens, num_heads, num_kv_heads, max_positions and num_pages must be positive")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim ({head_dim}) must be 64 or 128")
        if num_heads % self.num_kv_heads != 0:
            raise ValueError(f"num_heads ({num_heads}) must be divisible by num_kv_heads ({self.num_kv_heads})")
        if page_size < 64 or page_size & (page_size - 1):
            raise ValueError(f"page_size ({page_size}) must be a power of two >= 64")
        self.sections = (head_dim // 2,) if sections is None else tuple(int(n) for n in sections)
        if not 1 <= len(self.sections) <= 3 or min(self.sections) < 0 or sum(self.sections) != head_dim // 2:
            raise ValueError(f"sections {self.sections} must be one to three counts that add up to head_dim / 2 ({head_dim // 2})")
        self.interleaved = bool(interleaved)
        axes = len(self.sections)
        if self.interleaved and any(n and a + axes * (n - 1) >= head_dim // 2 for a, n in enumerate(self.sections) if a):
            raise ValueError(f"interleaved sections {self.sections} do not fit: axis a takes the frequencies a, a + {axes}, ...")
        self._backend = backend
        if backend == "ref":
            self._kernel = self._ref_forward
        else:
            self._kernel = get_kernel("paged_qk_norm_rope", backend)(
                num_heads, head_dim, max_positions, page_size, num_pages, num_kv_heads=self.num_kv_heads, sections=self.sections,
                interleaved=self.interleaved)

    def forward(self, qkv, q_norm_w, k_norm_w, cos, sin, positions, slots, K_pool, V_pool, out=None):
        return self._kernel(qkv, q_norm_w, k_norm_w, cos, sin, positions, slots, K_pool, V_pool, out)

    def check(self, actual, expected) -> bool:
        return actual.shape == expected.shape and torch.allclose(actual, expected, atol=self._atol, rtol=self._rtol)

    def rope_tables(self, device="cuda"):
        half = torch.arange(0, self.head_dim, 2, dtype=torch.float32, device=device) / self.head_dim
        ang = torch.arange(self.max_positions, dtype=torch.float32, device=device)[:, None] / self.rope_theta**half
        return tuple(torch.cat([f(ang)] * 2, dim=-1).to(torch.bfloat16) for f in (torch.cos, torch.sin))

    def gen_data(self, device="cuda"):
        kw = dict(device=device, dtype=torch.bfloat16)
        T, H, NKV, D = self.tokens, self.num_heads, self.num_kv_heads, self.head_dim
        qkv = torch.randn(T, (H + 2 * NKV) * D, **kw)
        q_norm_w, k_norm_w = torch.randn(D, **kw), torch.randn(D, **kw)
        cos, sin = self.rope_tables(device)
        axes = len(self.sections)
        positions = torch.randint(0, self.max_positions, (axes, T), dtype=torch.int32, device=device)
        slots = torch.randperm(self.num_pages * self.page_size, device=device)[:T].to(torch.int32)
        slots = torch.cat([slots, torch.full((T - slots.numel(),), -1, dtype=torch.int32, device=device)])
        K_pool, V_pool = (torch.randn(self.num_pages, NKV, self.page_size, D, **kw) for _ in range(2))
        return qkv, q_norm_w, k_norm_w, cos, sin, positions, slots, K_pool, V_pool

    def _ref_forward(self, qkv, q_norm_w, k_norm_w, cos, sin, positions, slots, K_pool, V_pool, out=None):
        T, H, NKV, D, page = qkv.shape[0], self.num_heads, self.num_kv_heads, self.head_dim, self.page_size
        positions = positions.reshape(len(self.sections), T).long()
        real = ((positions >= 0) & (positions < self.max_positions)).all(0)
        axis = torch.tensor(axis_of_frequency(self.sections, self.interleaved) * 2, device=qkv.device)
        at = positions.clamp(0, self.max_positions - 1)[axis].T  # [T, D]
        column = torch.arange(D, device=qkv.device)
        c, s = cos[at, column].float()[:, None], sin[at, column].float()[:, None]

        def head(x, w):
            n = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + self.rms_eps)
            if w is not None:
                n = n * w.float()
            rotated = torch.cat((-n[..., D // 2 :], n[..., : D // 2]), dim=-1)
            return (n * c + rotated * s).to(torch.bfloat16)

        x = qkv.float().view(T, H + 2 * NKV, D)
        q_out = torch.empty(T, H, D, dtype=torch.bfloat16, device=qkv.device) if out is None else out
        q_out[real] = head(x[:, :H], q_norm_w)[real]
        keep = real & (slots >= 0) & (slots < self.num_pages * page)
        slot = slots[keep].long()
        K_pool[slot // page, :, slot % page] = head(x[:, H : H + NKV], k_norm_w)[keep]
        V_pool[slot // page, :, slot % page] = x[:, H + NKV :].to(torch.bfloat16)[keep]
        return q_out
