"""The paged cache over libhkv (include/hkv.h, section "paged cache"): K/V rows of all requests in one pool of pages,
block tables and slot maps built on the GPU, append / norm + rotary positions through the slot map, attention of ragged
batches over the pages, cross attention to cached states.

PyTorch is used only for device memory and streams; all compute is in libhkv's kernels. Tensors are checked (type,
device, shape, strides) before a pointer is passed on; a wrong one raises HkvError with the status the library uses.
"""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass

from . import _capi
from ._capi import HkvError, HkvPagedGeometry, HkvPagedRope
from .ops import _ptr, _stream

_DTYPES = {"float16": 0, "bfloat16": 1}


def _dtype_code(dtype) -> int:
    name = str(dtype).replace("torch.", "")
    if name not in _DTYPES:
        raise HkvError(1, f"dtype {dtype}: the paged cache holds float16 or bfloat16")
    return _DTYPES[name]


@dataclass
class PagedGeometry:
    """Python view of `hkv_paged_geometry`."""
    num_heads: int = 32
    num_kv_heads: int | None = None
    head_dim: int = 128
    page_size: int = 16
    num_pages: int = 0
    max_requests: int = 1
    max_pages: int = 0          # columns of the block table = pages one request may hold
    max_tokens: int = 1         # packed tokens of one call
    window_size: int = 0
    dtype: object = "float16"   # or "bfloat16" / the torch dtypes
    kernel_select: int = _capi.KERNEL_AUTO
    flags: int = 0              # FLAG_APPEND_ONLY

    def to_c(self) -> HkvPagedGeometry:
        g = HkvPagedGeometry()
        g.dtype = _dtype_code(self.dtype)
        g.num_heads = self.num_heads
        g.num_kv_heads = self.num_heads if self.num_kv_heads is None else self.num_kv_heads
        g.head_dim, g.page_size, g.num_pages = self.head_dim, self.page_size, self.num_pages
        g.max_requests, g.max_pages, g.max_tokens = self.max_requests, self.max_pages, self.max_tokens
        g.window_size, g.kernel_select, g.flags = self.window_size, self.kernel_select, self.flags
        return g

    @property
    def default_scale(self) -> float:
        return 1.0 / math.sqrt(float(self.head_dim))


@dataclass
class PagedStep:
    """The tables of one step, as hkv_paged_plan writes them (int32, on the GPU)."""
    q_start: object     # [requests + 1]
    step_len: object    # [requests]
    total_len: object   # [requests]
    slots: object       # [tokens]
    positions: object   # [tokens]
    free_left: object   # [1]


class PagedContext:
    """Owns one `hkv_paged_ctx` (attention workspace + status word). Its calls must be ordered on the GPU."""

    def __init__(self, geometry: PagedGeometry):
        self.lib = _capi.load()
        self.geometry = geometry
        self._g = geometry.to_c()
        handle = C.c_void_p()
        st = self.lib.hkv_paged_create(C.byref(handle), C.byref(self._g))
        self._h = handle
        if st != _capi.HKV_OK:
            msg = self.lib.hkv_paged_last_error(handle).decode() if handle else "allocation failed"
            self.close()
            raise HkvError(st, msg)
        import torch
        self._device = torch.device("cuda", torch.cuda.current_device())
        self._dtype = torch.float16 if self._g.dtype == 0 else torch.bfloat16

    def close(self):
        if getattr(self, "_h", None):
            self.lib.hkv_paged_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, st: int):
        if st != _capi.HKV_OK:
            raise HkvError(st, self.lib.hkv_paged_last_error(self._h).decode())

    @property
    def workspace_bytes(self) -> int:
        return self.lib.hkv_paged_workspace_bytes(self._h)

    def device_status(self, stream=None) -> int:
        out = C.c_int32(0)
        st = self.lib.hkv_paged_device_status(self._h, _stream(stream), C.byref(out))
        if st not in (_capi.HKV_OK, 8):
            self._check(st)
        return out.value

    # -- argument checks ------------------------------------------------------
    def _ints(self, name, t, at_least: int):
        import torch
        if t.dtype != torch.int32 or t.device != self._device or not t.is_contiguous() or t.numel() < at_least:
            raise HkvError(1, f"{name}: a contiguous int32 tensor of at least {at_least} elements on {self._device} is wanted, "
                              f"got {t.dtype} {tuple(t.shape)} on {t.device}")
        return t.data_ptr() or 4        # no elements: not null, and not used

    def _rows(self, name, t, heads: int, tokens: int | None = None) -> tuple[int, int]:
        """(pointer, token stride) of a [tokens, heads, head_dim] tensor whose tokens may lie apart."""
        hd = self.geometry.head_dim
        if t.dtype != self._dtype or t.device != self._device or t.dim() != 3 or tuple(t.shape[1:]) != (heads, hd) or \
                (tokens is not None and t.shape[0] != tokens):
            raise HkvError(1, f"{name}: [{'tokens' if tokens is None else tokens}, {heads}, {hd}] {self._dtype} on {self._device} "
                              f"is wanted, got {tuple(t.shape)} {t.dtype} on {t.device}")
        if t.shape[0] == 0:
            return t.data_ptr() or 16, 0        # no rows: not null, and not used
        if (hd > 1 and t.stride(2) != 1) or (heads > 1 and t.stride(1) != hd):
            raise HkvError(2, f"{name}: heads and head_dim must be contiguous, strides {t.stride()}")
        return t.data_ptr(), (t.stride(0) if t.shape[0] > 1 else 0)

    def _plane(self, name, t):
        g = self.geometry
        want = (g.num_pages, g.page_size, self._g.num_kv_heads, g.head_dim)
        if t.dtype != self._dtype or t.device != self._device or tuple(t.shape) != want or not t.is_contiguous():
            raise HkvError(1, f"{name}: a contiguous {want} {self._dtype} plane on {self._device} is wanted, got "
                              f"{tuple(t.shape)} {t.dtype} on {t.device}")
        return t.data_ptr()

    def _table(self, t, requests: int):
        if t.dim() != 2 or t.shape[1] != self.geometry.max_pages:
            raise HkvError(1, f"block_table: [requests, {self.geometry.max_pages}] is wanted, got {tuple(t.shape)}")
        return self._ints("block_table", t, requests * self.geometry.max_pages)

    # -- tables ---------------------------------------------------------------
    def new_step(self, requests: int | None = None, tokens: int | None = None) -> PagedStep:
        """Tensors for the tables of one step (reused from step to step)."""
        import torch
        r = self.geometry.max_requests if requests is None else requests
        t = self.geometry.max_tokens if tokens is None else tokens
        make = lambda n: torch.zeros(n, dtype=torch.int32, device=self._device)
        return PagedStep(make(r + 1), make(r), make(r), make(t), make(t), make(1))

    def plan(self, past_len, new_len, block_table, free_pages, free_count, step: PagedStep, total_len=None, free_left=None,
             stream=None):
        """Block tables and slot maps of one step (hkv_paged_plan). `total_len=past_len, free_left=free_count` updates
        the state in place; by default both go to the step's own tensors."""
        r, t = past_len.numel(), step.slots.numel()
        total_len = step.total_len if total_len is None else total_len
        free_left = step.free_left if free_left is None else free_left
        self._check(self.lib.hkv_paged_plan(
            self._h, r, t, self._ints("past_len", past_len, r), self._ints("new_len", new_len, r), self._table(block_table, r),
            self._ints("free_pages", free_pages, self.geometry.num_pages), self._ints("free_count", free_count, 1),
            self._ints("total_len", total_len, r), self._ints("step_len", step.step_len, r),
            self._ints("q_start", step.q_start, r + 1), self._ints("slots", step.slots, t),
            self._ints("positions", step.positions, t), self._ints("free_left", free_left, 1), _stream(stream)))

    def release(self, finished, seq_len, block_table, free_pages, free_count, stream=None):
        """Gives the pages of the requests marked in `finished` back to the stack (hkv_paged_release)."""
        r = seq_len.numel()
        self._check(self.lib.hkv_paged_release(
            self._h, r, self._ints("finished", finished, r), self._ints("seq_len", seq_len, r), self._table(block_table, r),
            self._ints("free_pages", free_pages, self.geometry.num_pages), self._ints("free_count", free_count, 1),
            _stream(stream)))

    # -- rows into the pages ----------------------------------------------------
    def append(self, k_new, v_new, k_cache, v_cache, slots, stream=None):
        t = slots.numel()
        k, ks = self._rows("k_new", k_new, self._g.num_kv_heads, t)
        v, vs = self._rows("v_new", v_new, self._g.num_kv_heads, t)
        if ks != vs:
            raise HkvError(2, f"k_new and v_new have different token strides ({ks}, {vs})")
        self._check(self.lib.hkv_paged_append(self._h, k, v, ks, self._plane("k_cache", k_cache),
                                              self._plane("v_cache", v_cache), self._ints("slots", slots, t), t,
                                              _stream(stream)))

    def norm_rope(self, q, k, v, positions, slots=None, k_cache=None, v_cache=None, q_out=None, k_out=None, q_norm_w=None,
                  k_norm_w=None, sections=None, interleaved=False, rotary_dim=0, eps=1e-6, theta=10000.0,
                  scaling_factor=1.0, stream=None):
        """Per-head norm (with weights) + rotary positions with `positions` [axes, tokens] (or [tokens]); K and V to their
        slots when planes are given, else the turned k to `k_out` (default: in place). q_out defaults to q."""
        tokens, kvh, hd = q.shape[0], self._g.num_kv_heads, self.geometry.head_dim
        a = HkvPagedRope()
        a.q, a.q_token_stride = self._rows("q", q, self.geometry.num_heads)
        a.k, a.kv_token_stride = self._rows("k", k, kvh, tokens)
        a.q_out, a.q_out_token_stride = (a.q, a.q_token_stride) if q_out is None else \
            self._rows("q_out", q_out, self.geometry.num_heads, tokens)
        if k_cache is not None or v_cache is not None:
            if k_cache is None or v_cache is None or v is None or slots is None or k_out is not None:
                raise HkvError(1, "norm_rope: with cache planes both planes, v and slots are wanted and k_out is not")
            a.v, vs = self._rows("v", v, kvh, tokens)
            if vs != a.kv_token_stride:
                raise HkvError(2, f"k and v have different token strides ({a.kv_token_stride}, {vs})")
            a.k_cache, a.v_cache = self._plane("k_cache", k_cache), self._plane("v_cache", v_cache)
            a.d_slots = self._ints("slots", slots, tokens)
        else:
            a.k_out, a.k_out_token_stride = (a.k, a.kv_token_stride) if k_out is None else self._rows("k_out", k_out, kvh, tokens)
        for name, w in (("q_norm_w", q_norm_w), ("k_norm_w", k_norm_w)):
            if w is not None:
                if w.dtype != self._dtype or w.device != self._device or not w.is_contiguous() or w.numel() != hd:
                    raise HkvError(1, f"{name}: a contiguous [{hd}] {self._dtype} tensor on {self._device} is wanted")
                setattr(a, name, w.data_ptr())
        axes = 1 if positions.dim() == 1 else positions.shape[0]
        if positions.shape[-1] != tokens or positions.dim() > 2 or axes < 1:
            raise HkvError(1, f"positions: [axes, {tokens}] or [{tokens}] is wanted, got {tuple(positions.shape)}")
        a.d_positions = self._ints("positions", positions, axes * tokens)
        a.tokens, a.rotary_dim, a.axes, a.interleaved = tokens, rotary_dim, axes, int(bool(interleaved))
        sections = list(sections or [])
        if axes > 1 and (len(sections) != axes or axes > _capi.ROPE_MAX_AXES):
            raise HkvError(1, f"sections: one number per axis is wanted (at most {_capi.ROPE_MAX_AXES} axes), got {sections}")
        for i, s in enumerate(sections[:axes]):
            a.sections[i] = s
        a.eps, a.theta, a.scaling_factor = eps, theta, scaling_factor
        self._check(self.lib.hkv_paged_norm_rope(self._h, C.byref(a), _stream(stream)))

    # -- attention ---------------------------------------------------------------
    def _attend(self, fn, q, k_cache, v_cache, out, block_table, q_start, step_len, key_len, max_step, scale, stream):
        scale = self.geometry.default_scale if scale is None else scale
        r = key_len.numel()
        qp, qs = self._rows("q", q, self.geometry.num_heads)
        op, os_ = self._rows("out", out, self.geometry.num_heads, q.shape[0])
        if os_ not in (0, self.geometry.num_heads * self.geometry.head_dim):
            raise HkvError(2, f"out must be dense, token stride {os_}")
        self._check(fn(self._h, qp, qs, self._plane("k_cache", k_cache), self._plane("v_cache", v_cache), op,
                       self._table(block_table, r), self._ints("q_start", q_start, r), self._ints("step_len", step_len, r),
                       self._ints("key_len", key_len, r), r, q.shape[0], q.shape[0] if max_step is None else max_step, scale,
                       _stream(stream)))

    def attention(self, q, k_cache, v_cache, out, block_table, q_start, step_len, total_len, max_step=None, scale=None,
                  stream=None):
        """Attention of the packed new tokens over their requests' pages (hkv_paged_attention). `max_step`: upper bound of
        step_len; None = the packed tokens."""
        self._attend(self.lib.hkv_paged_attention, q, k_cache, v_cache, out, block_table, q_start, step_len, total_len,
                     max_step, scale, stream)

    def cross_attention(self, q, k_cache, v_cache, out, block_table, q_start, step_len, key_len, max_step=None, scale=None,
                        stream=None):
        """Attention of the packed queries over ALL cached rows of their requests (hkv_paged_cross_attention)."""
        self._attend(self.lib.hkv_paged_cross_attention, q, k_cache, v_cache, out, block_table, q_start, step_len, key_len,
                     max_step, scale, stream)
