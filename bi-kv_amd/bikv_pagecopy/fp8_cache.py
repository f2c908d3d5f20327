"""A paged KV cache held in 8 bits: appending new tokens to it and attending over it.

K and V are e4m3 bytes with one fp32 scale for each (page, layer, head, K/V). The bytes and scales are the caller's
tensors; `FP8KVCache.pool` is a PagedKVPool over the same memory, so pages of the cache are gathered, scattered,
staged to the host and copied with their scales as those of any pool.

The reference keeps its cache in fp16 and attends through a library over page indices it makes up on the host
(Bi-KV/Model/qwen2.py:169-181, 393-472). Here a step is two calls per layer on the current stream,

    cache.append(layer, k, v, page_table, kv_lens, q_starts)
    out = cache.attend(layer, q, page_table, kv_lens, q_starts)

with the sequences described by device tensors, so that a captured graph replays with other lengths:

  page_table  [n_seqs, max_pages] int64 page ids; entries behind a sequence's last page are not read
  kv_lens     [n_seqs] int64 tokens of each sequence, the step's own included
  q_starts    [n_seqs + 1] int64: rows q_starts[b] .. q_starts[b+1] of q, k, v are sequence b's newest tokens, in
              order; None = one row per sequence
"""
import ctypes as C
import math
import struct
from typing import Optional, Sequence

import torch
from torch.autograd import forward_ad

from . import _lib
from .pool import PagedKVPool, current_raw_stream

_SEQ_BATCH = struct.Struct("=7q2i")          # bikv_seq_batch
_TYPES = {torch.bfloat16: _lib.T_BF16, torch.float16: _lib.T_FP16}


def _end(t: torch.Tensor) -> int:
    """Address behind the last element of a tensor that has one."""
    return t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _has_tangent(t: torch.Tensor) -> bool:
    """Whether t carries a tangent of forward-mode differentiation."""
    return forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled() and forward_ad.unpack_dual(t).tangent is not None


class FP8KVCache:
    """`payload` [layers, 2, pages, page_tokens, kv_heads, head_dim] float8_e4m3fn (or uint8 with the same bytes) and
    `scale` [layers, 2, pages, kv_heads] float32, both contiguous on one GPU. `from_planes` takes one tensor per plane."""

    def __init__(self, payload: torch.Tensor, scale: torch.Tensor):
        if payload.dim() != 6 or payload.shape[1] != 2:
            raise RuntimeError("payload must be [layers, 2, pages, page_tokens, kv_heads, head_dim]")
        if tuple(scale.shape) != (payload.shape[0], 2, payload.shape[2], payload.shape[4]):
            raise RuntimeError("scale must be [layers, 2, pages, kv_heads]")
        PagedKVPool._check_plane(payload)
        PagedKVPool._check_plane(scale)
        self._refuse_gradients((payload, scale))
        self._open([payload[l, k] for l in range(payload.shape[0]) for k in (0, 1)],
                   [scale[l, k] for l in range(payload.shape[0]) for k in (0, 1)])

    @classmethod
    def from_planes(cls, planes: Sequence[torch.Tensor], scale_planes: Sequence[torch.Tensor]):
        """planes[2*layer + kv] is [pages, page_tokens, kv_heads, head_dim], scale_planes likewise [pages, kv_heads]."""
        self = cls.__new__(cls)
        self._open(list(planes), list(scale_planes))
        return self

    def _open(self, planes, scales):
        self._h = None
        self._refuse_gradients(planes + scales)
        p0 = planes[0] if planes else None
        if p0 is None or len(planes) % 2 or len(scales) != len(planes):
            raise RuntimeError("a cache has a K and a V plane per layer, and a scale plane to each")
        for t in planes:
            PagedKVPool._check_plane(t)
            if t.dtype not in (torch.float8_e4m3fn, torch.uint8) or t.dtype != p0.dtype or t.dim() != 4 or t.shape != p0.shape or t.device != p0.device:
                raise RuntimeError("planes must be float8_e4m3fn (or uint8) tensors [pages, page_tokens, kv_heads, head_dim] of one shape on one device")
        for t in scales:
            PagedKVPool._check_plane(t)
            if t.dtype != torch.float32 or tuple(t.shape) != (p0.shape[0], p0.shape[2]) or t.device != p0.device:
                raise RuntimeError("scale planes must be float32 tensors [pages, kv_heads] on the planes' device")
        self.device = p0.device
        self.n_layers = len(planes) // 2
        self.n_pages, self.page_tokens, self.kv_heads, self.head_dim = p0.shape
        d = _lib.FP8CacheDesc()
        d.device = self._device_index = p0.device.index
        d.n_layers, d.kv_heads, d.head_dim, d.page_tokens, d.n_pages = self.n_layers, self.kv_heads, self.head_dim, self.page_tokens, self.n_pages
        d.token_stride_bytes = self.kv_heads * self.head_dim
        d.page_stride_bytes = self.page_tokens * d.token_stride_bytes
        d.scale_page_stride_bytes = 4 * self.kv_heads
        ptrs = (C.c_void_p * len(planes))(*[t.data_ptr() for t in planes])
        sptrs = (C.c_void_p * len(planes))(*[t.data_ptr() for t in scales])
        d.plane_base = C.cast(ptrs, C.POINTER(C.c_void_p))
        d.scale_plane_base = C.cast(sptrs, C.POINTER(C.c_void_p))
        h = C.c_void_p()
        _lib.check(_lib.load().bikv_fp8_cache_create(C.byref(d), C.byref(h)))
        self._h = h
        self._lib = _lib.load()
        self._default_scale = 1.0 / math.sqrt(self.head_dim)
        self._workspace = {}
        self.pool = PagedKVPool.from_planes(planes, scales)      # keeps the tensors alive, too

    @staticmethod
    def _refuse_gradients(tensors):
        if torch.is_grad_enabled() and any(t.requires_grad for t in tensors) or any(_has_tangent(t) for t in tensors):
            raise RuntimeError("a cache's payload and scale are written in place and record no gradient: detach them or make the cache under torch.no_grad()")

    # ---- arguments ----------------------------------------------------------------------------
    # A step calls these once per layer, so the checks are few expressions and what is wrong is found out afterwards.
    def _rows(self, name, t, heads):
        """Strides (row, head) of a [rows, heads, head_dim] tensor the kernels can read; raises for any other."""
        shape, stride = t.shape, t.stride()
        if (t.device != self.device or len(shape) != 3 or shape[2] != self.head_dim or (heads is not None and shape[1] != heads)
                or t.dtype not in _TYPES or stride[2] != 1 and t.numel()):
            if t.device != self.device:
                raise RuntimeError(f"{name} must be on the cache's device")
            if t.dtype not in _TYPES:
                raise RuntimeError(f"{name} must be bfloat16 or float16")
            if len(shape) != 3 or shape[2] != self.head_dim or (heads is not None and shape[1] != heads):
                raise RuntimeError(f"{name} must be [rows, {heads if heads is not None else 'heads'}, {self.head_dim}], got {list(shape)}")
            raise RuntimeError(f"{name}: the values of a head must be contiguous")
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{name} requires a gradient, and the cache's calls record none: detach it or call under torch.no_grad()")
        if _has_tangent(t):
            raise RuntimeError(f"{name} carries a forward-mode gradient, and the cache's calls record none: pass its primal")
        return stride

    def _batch(self, rows, page_table, kv_lens, q_starts):
        """The bikv_seq_batch of a call, as bytes; raises for arrays that are not what it says."""
        n_rows, dtype = rows.shape[0], rows.dtype
        shape, stride, lens_shape = page_table.shape, page_table.stride(), kv_lens.shape
        dev, i64 = self.device, torch.int64
        if (page_table.dtype != i64 or page_table.device != dev or len(shape) != 2 or stride[1] != 1 and shape[1] > 1
                or stride[0] < shape[1] and shape[0] > 1):
            self._refuse_array("page_table", page_table, 2)
            raise RuntimeError("page_table's rows must not overlap")
        if kv_lens.dtype != i64 or kv_lens.device != dev or len(lens_shape) != 1 or kv_lens.stride(0) != 1 and lens_shape[0] > 1:
            self._refuse_array("kv_lens", kv_lens, 1)
        n = lens_shape[0]
        if shape[0] != n:
            raise RuntimeError("page_table and kv_lens differ in their number of sequences")
        starts = 0
        if q_starts is not None:
            if q_starts.dtype != i64 or q_starts.device != dev or q_starts.dim() != 1 or q_starts.stride(0) != 1 and q_starts.shape[0] > 1:
                self._refuse_array("q_starts", q_starts, 1)
            if q_starts.shape[0] != n + 1:
                raise RuntimeError("q_starts must have one entry more than there are sequences")
            starts = q_starts.data_ptr()
        elif n_rows != n:
            raise RuntimeError(f"without q_starts every sequence has one row: {n_rows} rows, {n} sequences")
        return _SEQ_BATCH.pack(page_table.data_ptr(), stride[0] if stride[0] > shape[1] else shape[1], shape[1], kv_lens.data_ptr(), starts, n, n_rows,
                               _TYPES[dtype], 0)

    def _refuse_array(self, name, t, dim):
        if t.device != self.device or t.dtype != torch.int64 or t.dim() != dim:
            raise RuntimeError(f"{name} must be a {dim}-D int64 tensor on the cache's device")
        if t.stride(-1) != 1 and t.shape[-1] > 1:
            raise RuntimeError(f"{name} must be contiguous along its last dimension")

    # ---- the two calls ------------------------------------------------------------------------
    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
               q_starts: Optional[torch.Tensor] = None):
        """Quantises k and v [rows, kv_heads, head_dim] (bf16 or fp16) into the pages of the sequences' last tokens, on the
        current stream (asynchronous). A page whose first token is new takes the smallest power-of-two scale that holds
        its new values; a page with older tokens keeps its scale as long as the new values fit, and is rounded to
        a larger one when they do not. A page may be written by one sequence of a call only (fork a shared last
        page with PagedKVPool.copy_pages first)."""
        ks, vs = self._rows("k", k, self.kv_heads), self._rows("v", v, self.kv_heads)
        if k.shape != v.shape or k.dtype != v.dtype:
            raise RuntimeError("k and v must share shape and dtype")
        batch = self._batch(k, page_table, kv_lens, q_starts)
        rc = self._lib.bikv_fp8_append(self._h, layer, batch, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1],
                                       current_raw_stream(self._device_index))
        if rc < 0:
            _lib.check(rc)

    def attend(self, layer: int, q: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
               q_starts: Optional[torch.Tensor] = None, causal: bool = True, softmax_scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None, return_lse: bool = False):
        """softmax(softmax_scale q K^T) V for q [rows, q_heads, head_dim] (bf16 or fp16) over each sequence's cached tokens,
        on the current stream (asynchronous); softmax_scale defaults to 1/sqrt(head_dim). With `causal` row t of a
        sequence's n rows sees the tokens up to its own (kv_len - n + t + 1 of them), without it all kv_len. Rows that see
        nothing get zeros (lse -inf). Returns out, or (out, lse) with lse [rows, q_heads] float32, the natural
        logarithm of the softmax's sum (what results over different pages are merged by). Rows behind the last
        sequence's are not written: in an `out` (and lse) made here they hold whatever the memory held. `out` must lie in
        other memory than q."""
        qs, shape = self._rows("q", q, None), q.shape
        batch = self._batch(q, page_table, kv_lens, q_starts)
        if out is None:
            out = q.new_empty(shape)
            os = out.stride()
        else:
            os = self._rows("out", out, None)
            if out.shape != shape or out.dtype != q.dtype:
                raise RuntimeError("out must have q's shape and dtype")
            (s0, s1, _), (n0, n1, _) = os, shape
            if out.numel() and not ((n1 == 1 or s1 >= self.head_dim) and (n0 == 1 or s0 >= s1 * (n1 - 1) + self.head_dim) or
                                    (n0 == 1 or s0 >= self.head_dim) and (n1 == 1 or s1 >= s0 * (n0 - 1) + self.head_dim)):
                raise RuntimeError("out's rows overlap")
            if out.numel() and out.data_ptr() < _end(q) and q.data_ptr() < _end(out):
                raise RuntimeError("out must not share memory with q")
        heads = shape[1]
        lse = q.new_empty(shape[:2], dtype=torch.float32) if return_lse else None
        key = (shape[0], heads, page_table.shape, q_starts is None)
        need = self._workspace.get(key)
        if need is None:                     # a size that follows from these numbers alone
            need = _lib.check(self._lib.bikv_fp8_attend_workspace(self._h, batch, heads))
            if len(self._workspace) >= 1024:
                self._workspace.clear()
            self._workspace[key] = need
        # from torch's allocator on the current stream: a call in flight elsewhere, or in another graph, has another one
        ws = q.new_empty(need // 2) if need else None
        rc = self._lib.bikv_fp8_attend(
            self._h, layer, batch, q.data_ptr(), qs[0], qs[1], heads, 1 if causal else 0,
            self._default_scale if softmax_scale is None else softmax_scale, out.data_ptr(), os[0], os[1],
            lse.data_ptr() if return_lse else None, ws.data_ptr() if need else None, need, current_raw_stream(self._device_index))
        if rc < 0:
            _lib.check(rc)
        return (out, lse) if return_lse else out

    def check(self):
        """Synchronises the current stream and raises if a kernel skipped a sequence or a page id."""
        self.pool.check()

    def close(self):
        if getattr(self, "_h", None):
            _lib.load().bikv_fp8_cache_destroy(self._h)
            self._h = None
        if getattr(self, "pool", None) is not None:
            self.pool.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
