"""The sm_100a backends of the prompt operators (see ``sm100.py`` for what all backends share).  They take any number of
tokens or rows per call, so the constructors hold what stays the same from step to step."""

from __future__ import annotations

import ctypes

import torch

from .. import _lib
from ..registry import register_kernel
from .base_kernel import BaseKernel
from .sm100 import _BF16, _current_device, _require, _stream, _zeros_bytes

_I32 = torch.int32


def _require_rows(t: torch.Tensor, name: str, shape, dtype=_BF16) -> int:
    """As ``_require``, but rows (the first dimension) may lie further apart; returns their distance in elements."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.numel() == 0:
        raise ValueError(f"{name} is empty")
    if t.is_contiguous():
        return t.numel() // t.shape[0]
    if not t[0].is_contiguous():
        raise ValueError(f"{name} must be contiguous within a row")
    return t.stride(0)


def _require_here(*tensors) -> None:
    """Launches go to the current device's current stream: tensors of another device do not belong there."""
    here = _current_device()
    for t in tensors:
        if t is not None and t.get_device() != here:
            raise ValueError(f"tensors are on {t.device}, but the current device is cuda:{here} (use torch.cuda.device)")


def _ptr(t):
    return None if t is None else t.data_ptr()


@register_kernel("paged_plan", "cuda", family="prompt")
class PagedPlanSm100Kernel(BaseKernel):
    def __init__(self, batch, max_tokens, max_pages, page_size, num_pages):
        if batch > 8192:
            raise ValueError(f"batch ({batch}) must be at most 8192")
        self.sizes = (batch, max_tokens, max_pages, page_size, num_pages)
        self._in = (("ctx_lens", (batch,)), ("new_lens", (batch,)), ("page_table", (batch, max_pages)))
        self._out = (("seq_lens", (batch,)), ("cu_tokens", (batch + 1,)), ("positions", (max_tokens,)), ("slots", (max_tokens,)),
                     ("free_count", (1,)))
        self._lib = _lib.load()

    def __call__(self, ctx_lens, new_lens, page_table, free_pages, free_count, out) -> None:
        for (name, shape), t in zip(self._in, (ctx_lens, new_lens, page_table)):
            _require(t, name, shape, _I32)
        _require(free_pages, "free_pages", (free_pages.numel(),), _I32)
        _require(free_count, "free_count", (1,), _I32)
        for (name, shape), t in zip(self._out, out):
            _require(t, f"out.{name}", shape, _I32)
        _require_here(ctx_lens, new_lens, page_table, free_pages, free_count, *out)
        _lib.check(self._lib.ezb_paged_plan(
            ctx_lens.data_ptr(), new_lens.data_ptr(), page_table.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(),
            *(t.data_ptr() for t in out), *self.sizes, free_pages.numel(), _stream()))


@register_kernel("paged_qk_norm_rope", "cuda", family="prompt")
class PagedQkNormRopeSm100Kernel(BaseKernel):
    rms_eps = 1e-6

    def __init__(self, num_heads, head_dim, max_positions, page_size, num_pages, num_kv_heads=None, sections=None, interleaved=False):
        self.H, self.D, self.S, self.P, self.pages = num_heads, head_dim, max_positions, page_size, num_pages
        self.NKV = num_heads if num_kv_heads is None else num_kv_heads
        self.sections = (head_dim // 2,) if sections is None else tuple(sections)
        self.interleaved = int(interleaved)
        self._sections = (ctypes.c_int * len(self.sections))(*self.sections)
        self._lib = _lib.load()

    def __call__(self, qkv, q_norm_w, k_norm_w, cos, sin, positions, slots, K_pool, V_pool, out=None):
        T, H, NKV, D, axes = qkv.shape[0], self.H, self.NKV, self.D, len(self.sections)
        ld = _require_rows(qkv, "qkv", (T, (H + 2 * NKV) * D))
        for name, t in (("q_norm_w", q_norm_w), ("k_norm_w", k_norm_w)):
            if t is not None:
                _require(t, name, (D,))
        _require(cos, "cos", (self.S, D)); _require(sin, "sin", (self.S, D))
        _require(positions, "positions", (T,) if axes == 1 and positions.dim() == 1 else (axes, T), _I32)
        _require(slots, "slots", (T,), _I32)
        pool = (self.pages, NKV, self.P, D)
        _require(K_pool, "K_pool", pool); _require(V_pool, "V_pool", pool)
        if out is None:
            out = torch.empty(T, H, D, dtype=_BF16, device=qkv.device)
        else:
            _require(out, "out", (T, H, D))
        _require_here(qkv, q_norm_w, k_norm_w, cos, sin, positions, slots, K_pool, V_pool, out)
        _lib.check(self._lib.ezb_paged_qk_norm_rope(
            qkv.data_ptr(), ld, _ptr(q_norm_w), _ptr(k_norm_w), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(), slots.data_ptr(),
            K_pool.data_ptr(), V_pool.data_ptr(), out.data_ptr(), T, H, NKV, D, self.S, axes, self._sections, self.interleaved, self.P,
            self.pages, self.rms_eps, _stream()))
        return out


@register_kernel("linear", "cuda", family="prompt")
class LinearSm100Kernel(BaseKernel):
    def __init__(self, out_features, in_features, bias=False, activation=None, residual=False, out_dtype=_BF16):
        from ..ops.linear import ACTIVATIONS

        if in_features % 8:
            raise ValueError(f"in_features ({in_features}) must be divisible by 8")
        self.N, self.K, self.out_dtype, self.act = out_features, in_features, out_dtype, ACTIVATIONS[activation]
        self.rows = out_features * (2 if activation == "swiglu" else 1)
        self._lib = _lib.load()

    def __call__(self, X, W, bias=None, residual=None, out=None):
        M, N, K = X.shape[0], self.N, self.K
        ldx = _require_rows(X, "X", (M, K))
        _require(W, "W", (self.rows, K))
        if bias is not None:
            _require(bias, "bias", (self.rows,))
        ldres = N if residual is None else _require_rows(residual, "residual", (M, N))
        if out is None:
            out = torch.empty(M, N, dtype=self.out_dtype, device=X.device)
        ldout = _require_rows(out, "out", (M, N), self.out_dtype)
        _require_here(X, W, bias, residual, out)
        _lib.check(self._lib.ezb_linear_bf16(X.data_ptr(), ldx, W.data_ptr(), _ptr(bias), _ptr(residual), ldres, out.data_ptr(), ldout,
                                             M, N, K, self.act, int(self.out_dtype == torch.float32), _stream()))
        return out


@register_kernel("attn_prompt", "cuda", family="prompt")
class AttnPromptSm100Kernel(BaseKernel):
    """Owns a workspace per device; one operator serves one stream at a time."""

    def __init__(self, batch, num_heads, head_dim, max_pages, page_size, num_kv_heads=None):
        self.B, self.H, self.D, self.max_pages, self.P = batch, num_heads, head_dim, max_pages, page_size
        self.NKV = num_heads if num_kv_heads is None else num_kv_heads
        self._ws = None
        self._lib = _lib.load()

    def workspace(self, device):
        if self._ws is None or self._ws.device != device:
            self._ws = _zeros_bytes(self._lib.ezb_attn_prompt_workspace_bytes(self.D), device)
        return self._ws

    def __call__(self, Q, K_pool, V_pool, page_table, seq_lens, cu_tokens, out=None):
        T, H, NKV, D = Q.shape[0], self.H, self.NKV, self.D
        ldq = _require_rows(Q, "Q", (T, H, D))
        for name, t in (("K_pool", K_pool), ("V_pool", V_pool)):
            _require(t, name, (K_pool.shape[0], NKV, self.P, D))
        _require(page_table, "page_table", (self.B, self.max_pages), _I32)
        _require(seq_lens, "seq_lens", (self.B,), _I32)
        _require(cu_tokens, "cu_tokens", (self.B + 1,), _I32)
        if out is None:
            out = torch.empty(T, H, D, dtype=_BF16, device=Q.device)
        ldo = _require_rows(out, "out", (T, H, D))
        _require_here(Q, K_pool, V_pool, page_table, seq_lens, cu_tokens, out)
        ws = self.workspace(Q.device)
        _lib.check(self._lib.ezb_attn_prompt(
            Q.data_ptr(), ldq, K_pool.data_ptr(), V_pool.data_ptr(), page_table.data_ptr(), seq_lens.data_ptr(), cu_tokens.data_ptr(),
            out.data_ptr(), ldo, ws.data_ptr(), ws.numel(), self.B, T, H, NKV, D, self.max_pages, self.P, K_pool.shape[0], _stream()))
        return out
