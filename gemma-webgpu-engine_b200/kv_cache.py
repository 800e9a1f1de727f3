"""Paged key/value cache on the GPU: quantised as it is written, read back, attended over.

The caller owns the pools: ``k`` and ``v`` [pages, kv_heads, page_size, head_dim] (any strides
with contiguous, 16-byte aligned rows) of bfloat16, float8_e4m3fn or int8; 8-bit pools have
one float32 scale per page, head and token, [pages, kv_heads, page_size].  A slot is
page · page_size + offset; a sequence's cached token j lies in page page_table[b, j // page_size].
``stream`` of a call is a raw stream handle in place of torch's current stream; outputs that the call
allocates belong to the stream it runs on.
"""
from __future__ import annotations

import ctypes
import struct

from . import _lib
from .sampling import SamplerError

# gs_kv_rows and gs_attention_args, packed in one go (a field-wise fill of the ctypes structures costs
# the host more than the launch)
_KV_ROWS = struct.Struct("=2Q4qQqi4x")
_ATTENTION_ARGS = struct.Struct("=6Q7q6if4x")


class GpuKvCache:
    """A handle on the pools (gs_kv_cache_create), on the sampler's context and device."""

    def __init__(self, sampler, k, v, k_scale=None, v_scale=None):
        import torch
        formats = {torch.bfloat16: _lib.GS_DTYPE_BF16, torch.float8_e4m3fn: _lib.GS_DTYPE_E4M3,
                   torch.int8: _lib.GS_DTYPE_INT8}
        if k.dtype not in formats or v.dtype != k.dtype:
            raise ValueError("k and v must both be bfloat16, float8_e4m3fn or int8")
        if k.dim() != 4 or v.shape != k.shape:
            raise ValueError("k and v must be [pages, kv_heads, page_size, head_dim]")
        self._device = torch.device("cuda", sampler.device)
        pages, heads, page_size, dim = k.shape
        quant = k.dtype != torch.bfloat16
        if quant != (k_scale is not None) or quant != (v_scale is not None):
            raise ValueError("k_scale and v_scale go with the 8-bit types")
        for t, what in ((k, "k"), (v, "v"), (k_scale, "k_scale"), (v_scale, "v_scale")):
            if t is not None and t.device != self._device:
                raise ValueError(f"{what} must be on the sampler's device")
        for t in (k, v):
            if t.stride(3) != 1:
                raise ValueError("rows of head_dim must be contiguous")
        for t in (k_scale, v_scale):
            if t is not None and (t.dtype != torch.float32 or tuple(t.shape) != (pages, heads, page_size) or
                                  not t.is_contiguous()):
                raise ValueError("scales must be contiguous float32 [pages, kv_heads, page_size]")
        self._L = _lib.lib()
        self._torch = torch
        self._sampler = sampler  # (keeps the context alive: its workspace serves the calls)
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.kv_heads, self.page_size, self.head_dim = pages, heads, page_size, dim
        d = _lib.GsKvCacheDesc()
        d.k, d.v = k.data_ptr(), v.data_ptr()
        if quant:
            d.k_scale, d.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
        d.pages, d.page_size, d.kv_heads, d.head_dim, d.format = pages, page_size, heads, dim, formats[k.dtype]
        d.k_page_stride, d.k_head_stride, d.k_token_stride = k.stride()[:3]
        d.v_page_stride, d.v_head_stride, d.v_token_stride = v.stride()[:3]
        self._int32, self._bf16 = torch.int32, torch.bfloat16
        self._types = {torch.bfloat16: _lib.GS_DTYPE_BF16, torch.float32: _lib.GS_DTYPE_F32}
        self._h = ctypes.c_void_p()
        if not sampler.handle:
            raise ValueError("the sampler is closed")
        st = self._L.gs_kv_cache_create(sampler.handle, ctypes.byref(d), ctypes.byref(self._h))
        if st != _lib.GS_OK:
            msg = sampler.last_error()
            raise ValueError(msg) if st == _lib.GS_EINVAL else SamplerError(st, msg)

    @classmethod
    def allocate(cls, sampler, pages: int, kv_heads: int, page_size: int, head_dim: int, format: str = "bf16"):
        """A cache of zeroed pools of its own (``format``: "bf16", "e4m3" or "int8")."""
        import torch
        types = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
        if format not in types:
            raise ValueError(f"format must be one of {sorted(types)}")
        dev = torch.device("cuda", sampler.device)
        shape = (pages, kv_heads, page_size, head_dim)
        k, v = (torch.zeros(shape, dtype=types[format], device=dev) for _ in range(2))
        scales = [torch.zeros(shape[:3], dtype=torch.float32, device=dev) if format != "bf16" else None for _ in range(2)]
        return cls(sampler, k, v, *scales)

    def close(self):
        if self._h:
            self._L.gs_kv_cache_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _fail(self, st):
        msg = (self._L.gs_kv_cache_last_error(self._h) or b"").decode()
        raise ValueError(msg) if st == _lib.GS_EINVAL else SamplerError(st, msg)

    def _open(self):
        # (the attention workspace is the context's: a closed sampler has given it back)
        if not self._h or not self._sampler.handle:
            raise ValueError("the cache or its sampler is closed")
        return self._h

    def _index(self, t, what, dims):
        if t.dtype is not self._int32 or t.dim() != dims or t.get_device() != self._sampler.device:
            raise ValueError(f"{what} must be an int32 tensor of {dims} dimension(s) on the sampler's device")
        if not t.is_contiguous() and t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{what} must be contiguous")

    def _move(self, call, k, v, slots, stream):
        self._index(slots, "slots", 1)
        dtype = self._types.get(k.dtype)
        if dtype is None or v.dtype is not k.dtype:
            raise ValueError("k and v must both be float32 or bfloat16")
        n = slots.shape[0]
        shape, dev = (n, self.kv_heads, self.head_dim), self._sampler.device
        k0, k1, k2 = k.stride() if k.dim() == 3 else (0, 0, 0)
        v0, v1, v2 = v.stride() if v.dim() == 3 else (0, 0, 0)
        if k.shape != shape or v.shape != shape or k2 != 1 or v2 != 1 or k.get_device() != dev or v.get_device() != dev:
            raise ValueError(f"k and v must be {list(shape)} with contiguous rows on the sampler's device")
        st = call(self._open(), _lib.pack_args(_KV_ROWS, k.data_ptr(), v.data_ptr(), k0, k1, v0, v1, slots.data_ptr(), n, dtype),
                  _lib.current_stream(self._device) if stream is None else stream)
        if st != _lib.GS_OK:
            self._fail(st)

    def write(self, k, v, slots, stream=None):
        """New keys and values [tokens, kv_heads, head_dim] (float32 or bfloat16) to ``slots``
        (int32 [tokens]; negative: skipped)."""
        self._move(self._L.gs_kv_write, k, v, slots, stream)

    def _new(self, slots, dtype):
        heads, dim = self.kv_heads, self.head_dim
        t = self._torch.bfloat16 if dtype is None else dtype
        k = self._torch.empty_strided((slots.shape[0], heads, dim), (heads * dim, dim, 1), dtype=t, device=self._device)
        return k, self._torch.empty_like(k)

    def read(self, slots, out=None, dtype=None, stream=None):
        """(k, v) [tokens, kv_heads, head_dim] at ``slots`` as ``dtype`` (bfloat16, or float32)."""
        if out is None:
            if stream is None:
                out = self._new(slots, dtype)
            else:
                with _lib.on_stream(stream, self._device):
                    out = self._new(slots, dtype)
        self._move(self._L.gs_kv_read, out[0], out[1], slots, stream)
        return out

    def attend(self, q, q_start, kv_len, page_table, *, max_kv: int, scale: float, max_q: int = 1, window: int = 0,
               sinks: int = 0, lse: bool = False, out=None, lse_out=None, stream=None):
        """Attention of the new tokens q [tokens, q_heads, head_dim] bfloat16 over the cache:
        sequence b has tokens [q_start[b], q_start[b + 1]) (None: one each) and kv_len[b] cached
        tokens, its new ones last.  ``window`` > 0: a token sees the last ``window`` positions and
        the first ``sinks``.  Returns (out like q, log-sum-exp [tokens, q_heads] or None)."""
        torch, dim, dev = self._torch, self.head_dim, self._sampler.device
        if q.dtype is not self._bf16 or q.dim() != 3 or q.shape[2] != dim or q.get_device() != dev:
            raise ValueError(f"q must be bfloat16 [tokens, q_heads, {dim}] on the sampler's device")
        tokens, heads, _ = q.shape
        # (a stride over a single token or head is never used: it is set to one that passes the checks)
        qt, qh, qd = q.stride()
        qt, qh = qt if tokens > 1 else heads * dim, qh if heads > 1 else dim
        if qd != 1:
            raise ValueError("q rows must be contiguous")
        self._index(kv_len, "kv_len", 1)
        self._index(page_table, "page_table", 2)
        seqs = kv_len.shape[0]
        rows, cols = page_table.shape
        if rows != seqs:
            raise ValueError("page_table must have one row per sequence")
        starts = 0
        if q_start is not None:
            self._index(q_start, "q_start", 1)
            if q_start.shape[0] != seqs + 1:
                raise ValueError("q_start must hold one entry more than kv_len")
            starts = q_start.data_ptr()
        if stream is not None and (out is None or (lse and lse_out is None)):
            with _lib.on_stream(stream, self._device):
                out = torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else out
                if lse and lse_out is None:
                    lse_out = torch.empty((tokens, heads), dtype=torch.float32, device=self._device)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            ot, oh = heads * dim, dim
        else:
            if out.dtype is not self._bf16 or out.shape != q.shape or out.stride(2) != 1 or out.get_device() != dev:
                raise ValueError("out must be bfloat16 of q's shape with contiguous rows on the sampler's device")
            ot = out.stride(0) if tokens > 1 else heads * dim
            oh = out.stride(1) if heads > 1 else dim
        if lse_out is not None:
            if lse_out.dtype != torch.float32 or lse_out.shape != (tokens, heads) or not lse_out.is_contiguous() or \
                    lse_out.get_device() != dev:
                raise ValueError("lse_out must be contiguous float32 [tokens, q_heads] on the sampler's device")
        elif lse:
            lse_out = torch.empty_strided((tokens, heads), (heads, 1), dtype=torch.float32, device=self._device)
        st = self._L.gs_attention(
            self._open(), _lib.pack_args(
                _ATTENTION_ARGS, q.data_ptr(), out.data_ptr(), lse_out.data_ptr() if lse_out is not None else 0, starts, kv_len.data_ptr(),
                page_table.data_ptr(), tokens, qt, qh, ot, oh, page_table.stride(0) if seqs > 1 else cols, cols, seqs, heads,
                max_q, max_kv, window, sinks, scale),
            _lib.current_stream(self._device) if stream is None else stream)
        if st != _lib.GS_OK:
            self._fail(st)
        return out, lse_out

    def check(self):
        """Raises when a kernel met a bad slot, page-table entry or length since the last check
        (synchronises)."""
        bits = ctypes.c_int32()
        st = self._L.gs_kv_cache_check(self._open(), ctypes.byref(bits))
        if st != _lib.GS_OK:
            self._fail(st)
