"""The sm_100a backends of the prompt operators (see ``sm100.py`` for what all backends share).  They take any number of
tokens or rows per call, so the constructors hold what stays the same from step to step."""

from __future__ import annotations

import ctypes
import struct

import torch

from .. import _lib
from ..registry import register_kernel
from .base_kernel import BaseKernel
from .sm100 import _BF16, _current_device, _raw_stream

_I32 = torch.int32
_capturing = torch.cuda.is_current_stream_capturing


# A step is a few short kernels, so the host's share counts (see sm100.py): a call asks everything about its tensors in one
# expression (0.2 us a tensor) and looks for what is wrong only when it fails.  Launches go to the current device's current
# stream, so tensors of another device are refused.
def _whole(t: torch.Tensor, shape, dtype, device: int) -> bool:
    return t.get_device() == device and t.dtype is dtype and t.shape == shape and t.is_contiguous()


def _rows(t: torch.Tensor, shape, dtype, device: int) -> bool:
    """As ``_whole``, but rows (the first dimension) may lie further apart."""
    return (t.get_device() == device and t.dtype is dtype and t.shape == shape and t.numel() > 0
            and (t.is_contiguous() or t[0].is_contiguous()))


def _device(t: torch.Tensor, name: str) -> int:
    """The current device, if there is one."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return _current_device()


def _refuse(checks, device: int, no_rows: bool = False):
    """Raises for the first of ``checks`` - (name, tensor, shape, dtype, rows may lie apart) - that does not hold.  It returns when
    all hold but for tensors that are empty because the call has ``no_rows``: then there is nothing to do."""
    for name, t, shape, dtype, apart in checks:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor")
        if t.get_device() != device:
            raise ValueError(f"{name} is on {t.device}, but the current device is cuda:{device} (use torch.cuda.device)")
        if t.dtype != dtype:
            raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
        if tuple(t.shape) != tuple(shape):
            raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
        if t.numel() == 0 and not no_rows:
            raise ValueError(f"{name} is empty")
        if not t.is_contiguous() and not (apart and t[0].is_contiguous()):
            raise ValueError(f"{name} must be contiguous" + (" within a row" if apart else ""))


def _distance(t: torch.Tensor) -> int:
    """Elements from one row to the next."""
    return t.numel() // t.shape[0] if t.is_contiguous() else t.stride(0)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _packed(entry: str):
    """The packed form of a C entry (its arguments as 64-bit words in one bytes object) and what packs them: ctypes converts one
    argument instead of twenty."""
    words = len(_lib.SIGNATURES[entry][1])
    return getattr(_lib.load(), entry + "_packed"), struct.Struct(f"{words}q").pack


class _Workspaces:
    """The workspaces of one operator: one per device and stream, and one per stream of a graph capture, so that neither calls on
    several streams nor graphs that are replayed side by side meet in one.  A captured call never uses an eager one's, nor the
    other way round: the counters in front (all that has to be zero) are cleared where the memory is first used, in a graph
    once per replay.  A capture's are dropped when the next one begins: they lie in its graph's own pool.

    A call that gives up a wait leaves its counters half counted.  Once ``_lib.device_status`` has read a fault (any: the word
    keeps the first one only), the eager workspaces are dropped, and calls go on with cleared ones."""

    _COUNTERS = 4096
    _STREAMS = 8  # eager ones that are kept: of more streams the oldest one's goes (its memory is reused behind its stream's work)

    def __init__(self, lib):
        self._lib, self._eager, self._captured, self._capture, self._faults = lib, {}, {}, 0, _lib.faults_read

    def get(self, nbytes: int, device: int, stream: int):
        held = self._eager
        if _capturing():
            capture = self._lib.ezb_stream_capture_id(stream)
            if capture != self._capture:
                self._capture, self._captured = capture, {}
            held = self._captured
        elif self._faults != _lib.faults_read:
            self._faults = _lib.faults_read
            held.clear()
        ws = held.get((device, stream))
        if ws is None:
            if held is self._eager and len(held) >= self._STREAMS:
                held.pop(list(held)[0], None)
            ws = held[device, stream] = torch.empty(nbytes, dtype=torch.uint8, device=torch.device("cuda", device))
            ws[: self._COUNTERS].zero_()
        return ws


@register_kernel("paged_plan", "cuda", family="prompt")
class PagedPlanSm100Kernel(BaseKernel):
    def __init__(self, batch, max_tokens, max_pages, page_size, num_pages):
        if batch > 8192:
            raise ValueError(f"batch ({batch}) must be at most 8192")
        self.sizes = (batch, max_tokens, max_pages, page_size, num_pages)
        self._rows, self._table, self._cu, self._tokens, self._one = (batch,), (batch, max_pages), (batch + 1,), (max_tokens,), (1,)
        self._entry, self._pack = _packed("ezb_paged_plan")

    def __call__(self, ctx_lens, new_lens, page_table, free_pages, free_count, out) -> None:
        dev, rows, tokens, one = _device(ctx_lens, "ctx_lens"), self._rows, self._tokens, self._one
        lens, cu, positions, slots, left = out
        free = (free_pages.numel(),)
        if not (_whole(ctx_lens, rows, _I32, dev) and _whole(new_lens, rows, _I32, dev) and _whole(page_table, self._table, _I32, dev)
                and _whole(free_pages, free, _I32, dev) and _whole(free_count, one, _I32, dev) and _whole(lens, rows, _I32, dev)
                and _whole(cu, self._cu, _I32, dev) and _whole(positions, tokens, _I32, dev) and _whole(slots, tokens, _I32, dev)
                and _whole(left, one, _I32, dev) and free[0] > 0):
            _refuse([(n, t, shape, _I32, False) for n, t, shape in (
                ("ctx_lens", ctx_lens, rows), ("new_lens", new_lens, rows), ("page_table", page_table, self._table),
                ("free_pages", free_pages, free), ("free_count", free_count, one), ("out.seq_lens", lens, rows),
                ("out.cu_tokens", cu, self._cu), ("out.positions", positions, tokens), ("out.slots", slots, tokens),
                ("out.free_count", left, one))], dev)
        rc = self._entry(self._pack(
            ctx_lens.data_ptr(), new_lens.data_ptr(), page_table.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(),
            lens.data_ptr(), cu.data_ptr(), positions.data_ptr(), slots.data_ptr(), left.data_ptr(), *self.sizes, free[0],
            _raw_stream(dev)))
        if rc:
            _lib.check(rc)


@register_kernel("paged_qk_norm_rope", "cuda", family="prompt")
class PagedQkNormRopeSm100Kernel(BaseKernel):
    rms_eps = 1e-6

    def __init__(self, num_heads, head_dim, max_positions, page_size, num_pages, num_kv_heads=None, sections=None, interleaved=False):
        NKV = num_heads if num_kv_heads is None else num_kv_heads
        self.H, self.D = num_heads, head_dim
        sections = (head_dim // 2,) if sections is None else tuple(sections)
        self.axes = len(sections)
        self._sections = (ctypes.c_int * self.axes)(*sections)
        self._width, self._w, self._table = (num_heads + 2 * NKV) * head_dim, (head_dim,), (max_positions, head_dim)
        self._pool = (num_pages, NKV, page_size, head_dim)
        eps = struct.unpack("i", struct.pack("f", self.rms_eps))[0]
        self._sizes = (num_heads, NKV, head_dim, max_positions, self.axes, ctypes.addressof(self._sections), int(interleaved), page_size,
                       num_pages, eps)
        self._entry, self._pack = _packed("ezb_paged_qk_norm_rope")

    def __call__(self, qkv, q_norm_w, k_norm_w, cos, sin, positions, slots, K_pool, V_pool, out=None):
        dev, T, w, table, pool = _device(qkv, "qkv"), qkv.shape[0], self._w, self._table, self._pool
        row = (T, self._width)
        if out is None:
            out = torch.empty(T, self.H, self.D, dtype=_BF16, device=qkv.device)
        where = (T,) if self.axes == 1 and positions.dim() == 1 else (self.axes, T)
        heads = (T, self.H, self.D)
        if not (_rows(qkv, row, _BF16, dev) and (q_norm_w is None or _whole(q_norm_w, w, _BF16, dev))
                and (k_norm_w is None or _whole(k_norm_w, w, _BF16, dev)) and _whole(cos, table, _BF16, dev)
                and _whole(sin, table, _BF16, dev) and _whole(positions, where, _I32, dev) and _whole(slots, (T,), _I32, dev)
                and _whole(K_pool, pool, _BF16, dev) and _whole(V_pool, pool, _BF16, dev) and _whole(out, heads, _BF16, dev)):
            _refuse([("qkv", qkv, row, _BF16, True), ("q_norm_w", q_norm_w, w, _BF16, False), ("k_norm_w", k_norm_w, w, _BF16, False),
                     ("cos", cos, table, _BF16, False), ("sin", sin, table, _BF16, False), ("positions", positions, where, _I32, False),
                     ("slots", slots, (T,), _I32, False), ("K_pool", K_pool, pool, _BF16, False), ("V_pool", V_pool, pool, _BF16, False),
                     ("out", out, heads, _BF16, False)], dev, T == 0)
            if T == 0:
                return out
        rc = self._entry(self._pack(
            qkv.data_ptr(), _distance(qkv), _ptr(q_norm_w), _ptr(k_norm_w), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(),
            slots.data_ptr(), K_pool.data_ptr(), V_pool.data_ptr(), out.data_ptr(), T, *self._sizes, _raw_stream(dev)))
        if rc:
            _lib.check(rc)
        return out


@register_kernel("linear", "cuda", family="prompt")
class LinearSm100Kernel(BaseKernel):
    def __init__(self, out_features, in_features, bias=False, activation=None, residual=False, out_dtype=_BF16):
        from ..ops.linear import ACTIVATIONS

        if in_features % 8:
            raise ValueError(f"in_features ({in_features}) must be divisible by 8")
        self.N, self.K, self.out_dtype, self.act = out_features, in_features, out_dtype, ACTIVATIONS[activation]
        rows = out_features * (2 if activation == "swiglu" else 1)
        self._w, self._bias = (rows, in_features), (rows,)
        self._f32 = int(out_dtype == torch.float32)
        self._entry, self._pack = _packed("ezb_linear_bf16")

    def __call__(self, X, W, bias=None, residual=None, out=None):
        dev, M, N, K = _device(X, "X"), X.shape[0], self.N, self.K
        if out is None:
            out = torch.empty(M, N, dtype=self.out_dtype, device=X.device)
        if not (_rows(X, (M, K), _BF16, dev) and _whole(W, self._w, _BF16, dev) and (bias is None or _whole(bias, self._bias, _BF16, dev))
                and (residual is None or _rows(residual, (M, N), _BF16, dev)) and _rows(out, (M, N), self.out_dtype, dev)):
            _refuse([("X", X, (M, K), _BF16, True), ("W", W, self._w, _BF16, False), ("bias", bias, self._bias, _BF16, False),
                     ("residual", residual, (M, N), _BF16, True), ("out", out, (M, N), self.out_dtype, True)], dev, M == 0)
            if M == 0:
                return out
        rc = self._entry(self._pack(
            X.data_ptr(), _distance(X), W.data_ptr(), _ptr(bias), _ptr(residual), N if residual is None else _distance(residual),
            out.data_ptr(), _distance(out), M, N, K, self.act, self._f32, _raw_stream(dev)))
        if rc:
            _lib.check(rc)
        return out


@register_kernel("attn_prompt", "cuda", family="prompt")
class AttnPromptSm100Kernel(BaseKernel):
    """Owns workspaces (``_Workspaces``)."""

    def __init__(self, batch, num_heads, head_dim, max_pages, page_size, num_kv_heads=None):
        self.B, self.H, self.D, self.max_pages, self.P = batch, num_heads, head_dim, max_pages, page_size
        self.NKV = num_heads if num_kv_heads is None else num_kv_heads
        self._table, self._lens, self._cu = (batch, max_pages), (batch,), (batch + 1,)
        self._lib = _lib.load()
        self._entry, self._pack = _packed("ezb_attn_prompt")
        self._need = self._lib.ezb_attn_prompt_workspace_bytes(self.D)
        self._spaces = _Workspaces(self._lib)

    def __call__(self, Q, K_pool, V_pool, page_table, seq_lens, cu_tokens, out=None):
        dev, T, H, D = _device(Q, "Q"), Q.shape[0], self.H, self.D
        heads, pool = (T, H, D), (K_pool.shape[0], self.NKV, self.P, D)
        if out is None:
            out = torch.empty(T, H, D, dtype=_BF16, device=Q.device)
        if not (_rows(Q, heads, _BF16, dev) and _whole(K_pool, pool, _BF16, dev) and _whole(V_pool, pool, _BF16, dev)
                and _whole(page_table, self._table, _I32, dev) and _whole(seq_lens, self._lens, _I32, dev)
                and _whole(cu_tokens, self._cu, _I32, dev) and _rows(out, heads, _BF16, dev)):
            _refuse([("Q", Q, heads, _BF16, True), ("K_pool", K_pool, pool, _BF16, False), ("V_pool", V_pool, pool, _BF16, False),
                     ("page_table", page_table, self._table, _I32, False), ("seq_lens", seq_lens, self._lens, _I32, False),
                     ("cu_tokens", cu_tokens, self._cu, _I32, False), ("out", out, heads, _BF16, True)], dev, T == 0)
            if T == 0:
                return out
        stream = _raw_stream(dev)
        ws = self._spaces.get(self._need, dev, stream)
        rc = self._entry(self._pack(
            Q.data_ptr(), _distance(Q), K_pool.data_ptr(), V_pool.data_ptr(), page_table.data_ptr(), seq_lens.data_ptr(),
            cu_tokens.data_ptr(), out.data_ptr(), _distance(out), ws.data_ptr(), self._need, self.B, T, H, self.NKV, D, self.max_pages,
            self.P, pool[0], stream))
        if rc:
            _lib.check(rc)
        return out
