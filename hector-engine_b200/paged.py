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
_INT32 = None               # torch.int32, once a context exists


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
        global _INT32
        _INT32 = torch.int32
        self._index = torch.cuda.current_device()
        self._device = torch.device("cuda", self._index)
        self._dtype = torch.float16 if self._g.dtype == 0 else torch.bfloat16
        g = self._g
        self._heads, self._kvh, self._hd, self._cols = g.num_heads, g.num_kv_heads, g.head_dim, g.max_pages
        self._plane_shape = (g.num_pages, g.page_size, g.num_kv_heads, g.head_dim)
        # the raw handle of torch's current stream, without a Stream object per call
        self._current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
            (lambda index: torch.cuda.current_stream(index).cuda_stream)

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
        st = self.lib.hkv_paged_device_status(self._h, self._stream(stream), C.byref(out))
        if st not in (_capi.HKV_OK, 8):
            self._check(st)
        return out.value

    # -- argument checks ------------------------------------------------------
    # A decode step makes several of these calls per layer, so the checks are written for their cost: singletons are
    # compared by identity and an error's text is put together only when there is one.
    def _ints(self, name, t, at_least):
        n = t.numel()
        if t.dtype is not _INT32 or t.get_device() != self._index or n < at_least or not t.is_contiguous():
            raise HkvError(1, f"{name}: a contiguous int32 tensor of at least {at_least} elements on cuda:{self._index} is "
                              f"wanted, got {t.dtype} {tuple(t.shape)} on {t.device}")
        return t.data_ptr() if n else 4     # no elements: not null, and not used

    def _rows(self, name, t, heads, tokens):
        """(pointer, token stride) of a [tokens, heads, head_dim] tensor whose tokens may lie apart."""
        hd = self._hd
        if t.dtype is not self._dtype or t.get_device() != self._index or t.shape != (tokens, heads, hd):
            raise HkvError(1, f"{name}: [{tokens}, {heads}, {hd}] {self._dtype} on cuda:{self._index} is wanted, got "
                              f"{tuple(t.shape)} {t.dtype} on {t.device}")
        if t.is_contiguous():
            return (t.data_ptr() if tokens else 16), 0      # no rows: not null, and not used
        s = t.stride()
        if (hd > 1 and s[2] != 1) or (heads > 1 and s[1] != hd):
            raise HkvError(2, f"{name}: heads and head_dim must be contiguous, strides {s}")
        if tokens > 1 and s[0] < heads * hd:                # (a broadcast token's stride of 0 would mean "dense" below)
            raise HkvError(2, f"{name}: tokens overlap, strides {s}: expand()ed rows have to be copied first")
        return t.data_ptr(), (s[0] if tokens > 1 else 0)

    def _plane(self, name, t):
        if t.dtype is not self._dtype or t.get_device() != self._index or t.shape != self._plane_shape or not t.is_contiguous():
            raise HkvError(1, f"{name}: a contiguous {self._plane_shape} {self._dtype} plane on cuda:{self._index} is wanted, got "
                              f"{tuple(t.shape)} {t.dtype} on {t.device}")
        return t.data_ptr()

    def _table(self, t, requests):
        if t.dim() != 2 or t.shape[1] != self._cols:
            raise HkvError(1, f"block_table: [requests, {self._cols}] is wanted, got {tuple(t.shape)}")
        return self._ints("block_table", t, requests * self._cols)

    def _stream(self, stream):
        return self._current_stream(self._index) if stream is None else _stream(stream)

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
            self._ints("positions", step.positions, t), self._ints("free_left", free_left, 1), self._stream(stream)))

    def release(self, finished, seq_len, block_table, free_pages, free_count, stream=None):
        """Gives the pages of the requests marked in `finished` back to the stack (hkv_paged_release)."""
        r = seq_len.numel()
        self._check(self.lib.hkv_paged_release(
            self._h, r, self._ints("finished", finished, r), self._ints("seq_len", seq_len, r), self._table(block_table, r),
            self._ints("free_pages", free_pages, self.geometry.num_pages), self._ints("free_count", free_count, 1),
            self._stream(stream)))

    # -- rows into the pages ----------------------------------------------------
    def append(self, k_new, v_new, k_cache, v_cache, slots, stream=None):
        """K and V rows of the packed tokens to their slots (hkv_paged_append)."""
        t = slots.numel()
        k, ks = self._rows("k_new", k_new, self._kvh, t)
        v, vs = self._rows("v_new", v_new, self._kvh, t)
        if ks != vs:
            raise HkvError(2, f"k_new and v_new have different token strides ({ks}, {vs})")
        st = self.lib.hkv_paged_append(self._h, k, v, ks, self._plane("k_cache", k_cache), self._plane("v_cache", v_cache),
                                       self._ints("slots", slots, t), t, self._stream(stream))
        if st:
            self._check(st)

    def norm_rope(self, q, k, v, positions, slots=None, k_cache=None, v_cache=None, q_out=None, k_out=None, q_norm_w=None,
                  k_norm_w=None, sections=None, interleaved=False, rotary_dim=0, eps=1e-6, theta=10000.0,
                  scaling_factor=1.0, stream=None):
        """Per-head norm (with weights) + rotary positions with `positions` [axes, tokens] (or [tokens]); K and V to their
        slots when planes are given, else the turned k to `k_out` (default: in place). q_out defaults to q."""
        tokens, kvh, hd = q.shape[0], self._kvh, self._hd
        a = HkvPagedRope()
        a.q, a.q_token_stride = self._rows("q", q, self._heads, tokens)
        a.k, a.kv_token_stride = ks = self._rows("k", k, kvh, tokens)
        a.q_out, a.q_out_token_stride = self._rows("q_out", q if q_out is None else q_out, self._heads, tokens)
        if k_cache is not None or v_cache is not None:
            if k_cache is None or v_cache is None or v is None or slots is None or k_out is not None:
                raise HkvError(1, "norm_rope: with cache planes both planes, v and slots are wanted and k_out is not")
            a.v, vs = self._rows("v", v, kvh, tokens)
            if vs != ks[1]:
                raise HkvError(2, f"k and v have different token strides ({ks[1]}, {vs})")
            a.k_cache, a.v_cache = self._plane("k_cache", k_cache), self._plane("v_cache", v_cache)
            a.d_slots = self._ints("slots", slots, tokens)
        else:
            a.k_out, a.k_out_token_stride = self._rows("k_out", k if k_out is None else k_out, kvh, tokens)
        for name, w in (("q_norm_w", q_norm_w), ("k_norm_w", k_norm_w)):
            if w is not None:
                if w.dtype is not self._dtype or w.get_device() != self._index or w.numel() != hd or not w.is_contiguous():
                    raise HkvError(1, f"{name}: a contiguous [{hd}] {self._dtype} tensor on cuda:{self._index} is wanted")
                setattr(a, name, w.data_ptr())
        shape = positions.shape
        axes = shape[0] if len(shape) == 2 else 1
        if len(shape) not in (1, 2) or shape[-1] != tokens or axes < 1:
            raise HkvError(1, f"positions: [axes, {tokens}] or [{tokens}] is wanted, got {tuple(shape)}")
        a.d_positions = self._ints("positions", positions, axes * tokens)
        a.tokens, a.rotary_dim, a.axes, a.interleaved = tokens, rotary_dim, axes, 1 if interleaved else 0
        if axes > 1:
            if sections is None or len(sections) != axes or axes > _capi.ROPE_MAX_AXES:
                raise HkvError(1, f"sections: one number per axis is wanted (at most {_capi.ROPE_MAX_AXES} axes), got {sections}")
            a.sections[:axes] = sections
        a.eps, a.theta, a.scaling_factor = eps, theta, scaling_factor
        st = self.lib.hkv_paged_norm_rope(self._h, a, self._stream(stream))
        if st:
            self._check(st)

    # -- attention ---------------------------------------------------------------
    def _attend(self, fn, q, k_cache, v_cache, out, block_table, q_start, step_len, key_len, max_step, scale, stream):
        r, tokens = key_len.numel(), q.shape[0]
        qp, qs = self._rows("q", q, self._heads, tokens)
        op, os_ = self._rows("out", out, self._heads, tokens)
        if os_:
            raise HkvError(2, f"out must be dense, token stride {os_}")
        st = fn(self._h, qp, qs, self._plane("k_cache", k_cache), self._plane("v_cache", v_cache), op,
                self._table(block_table, r), self._ints("q_start", q_start, r), self._ints("step_len", step_len, r),
                self._ints("key_len", key_len, r), r, tokens, tokens if max_step is None else max_step,
                self.geometry.default_scale if scale is None else scale, self._stream(stream))
        if st:
            self._check(st)

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
