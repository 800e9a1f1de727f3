"""Residual + RMS norm with an 8-bit output (gs_rms_norm): the pass before a product.

Per row, in float32: h = x + residual, y = h · (mean(h²) + eps)^-1/2 · (weight_offset + weight);
h is kept for the next layer, y goes out as float32 / bfloat16, as e4m3 codes with a float32
scale per row or per group of columns, or (``srq_scale``) on the int8 grid that
``GpuLmHead`` reads, with its row sum.
"""
from __future__ import annotations

import struct
from dataclasses import dataclass

from . import _lib
from .sampling import SamplerError

_RMS_NORM_ARGS = struct.Struct("=7Q6q4i3f4x")  # gs_rms_norm_args


@dataclass(slots=True)
class RmsNormResult:
    out: object              # [rows, hidden] of the output type
    scale: object = None     # [rows, groups] float32 (e4m3)
    residual: object = None  # [rows, hidden] x + residual, of x's type (None without a residual)
    row_sum: object = None   # [rows] float32 (srq): the LM head's activation_sum


class GpuRmsNorm:
    """One norm's weight and output form on the sampler's device (``out``: "bf16", "f32",
    "e4m3", or "srq" with ``srq_scale``; ``group``: 0, 32, 64 or 128 columns per e4m3 scale)."""

    OUTS = ("bf16", "f32", "e4m3", "srq")

    def __init__(self, sampler, weight=None, *, hidden: int | None = None, eps: float = 1e-6, weight_offset: float = 0.0,
                 out: str = "bf16", group: int = 0, srq_scale: float = 0.0):
        import torch
        if out not in self.OUTS:
            raise ValueError(f"out must be one of {self.OUTS}")
        if (out == "srq") != (srq_scale != 0.0):
            raise ValueError("srq_scale goes with out='srq'")
        if weight is not None:
            if weight.dim() != 1 or weight.dtype not in (torch.float32, torch.bfloat16):
                raise ValueError("weight must be [hidden] float32 or bfloat16")
            if weight.device != torch.device("cuda", sampler.device):
                raise ValueError("weight must be on the sampler's device")
            weight = weight.contiguous()
            hidden = weight.shape[0]
        if hidden is None:
            raise ValueError("hidden or weight is required")
        self._L = _lib.lib()
        self._sampler = sampler  # (keeps the context alive)
        self.hidden, self.out, self.group, self._weight = int(hidden), out, int(group), weight
        self.groups = -(-self.hidden // self.group) if self.group else 1
        self._torch = torch
        self._device = torch.device("cuda", sampler.device)
        self._out_type = {"bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn,
                          "srq": torch.float32}[out]
        # gs_rms_norm_args is filled by one struct.pack a call: (pointers, sizes, types) around what is fixed
        self._weight_ptr = weight.data_ptr() if weight is not None else 0
        self._tail = (_lib.GS_DTYPE_BF16 if weight is not None and weight.dtype == torch.bfloat16 else _lib.GS_DTYPE_F32,
                      {"bf16": _lib.GS_DTYPE_BF16, "f32": _lib.GS_DTYPE_F32, "e4m3": _lib.GS_DTYPE_E4M3,
                       "srq": _lib.GS_DTYPE_F32}[out], self.group, float(eps), float(weight_offset), float(srq_scale))
        self._types = {torch.bfloat16: _lib.GS_DTYPE_BF16, torch.float32: _lib.GS_DTYPE_F32}

    def _stride(self, t, what, rows, dtype):
        if t.dtype is not dtype or t.get_device() != self._sampler.device or t.shape != (rows, self.hidden):
            raise ValueError(f"{what} must be {dtype} [{rows}, {self.hidden}] on the sampler's device")
        s0, s1 = t.stride()
        if s1 != 1 and self.hidden > 1:
            raise ValueError(f"{what} rows must be contiguous")
        return s0 if rows > 1 else self.hidden

    def _new(self, x, rows, with_residual):
        torch, dev = self._torch, self._device
        return RmsNormResult(
            torch.empty_like(x, dtype=self._out_type, memory_format=torch.contiguous_format),
            torch.empty_strided((rows, self.groups), (self.groups, 1), dtype=torch.float32, device=dev)
            if self.out == "e4m3" else None,
            torch.empty_like(x, memory_format=torch.contiguous_format) if with_residual else None,
            torch.empty(rows, dtype=torch.float32, device=dev) if self.out == "srq" else None)

    def __call__(self, x, residual=None, *, out: RmsNormResult | None = None, stream=None) -> RmsNormResult:
        """The norm of x (+ residual), both [rows, hidden] float32 or bfloat16.  ``out``: a result
        to write into (its ``residual`` may be the residual itself).  ``stream``: a raw stream handle in place of
        torch's current one; results allocated here then belong to that stream."""
        torch, hidden, xt = self._torch, self.hidden, x.dtype
        dtype = self._types.get(xt)
        if dtype is None:
            raise ValueError("x must be float32 or bfloat16")
        if x.dim() != 2:
            raise ValueError(f"x must be [rows, {hidden}]")
        rows = x.shape[0]
        ld_x = self._stride(x, "x", rows, xt)
        ld_r = self._stride(residual, "residual", rows, xt) if residual is not None else 0
        if out is None:
            if stream is None:
                out = self._new(x, rows, residual is not None)
            else:
                with _lib.on_stream(stream, self._device):
                    out = self._new(x, rows, residual is not None)
            ld_out = ld_ro = hidden
        else:
            ld_out = self._stride(out.out, "out.out", rows, self._out_type)
            ld_ro = self._stride(out.residual, "out.residual", rows, xt) if out.residual is not None else 0
            for t, shape in ((out.scale, (rows, self.groups)), (out.row_sum, (rows,))):
                if t is not None and (t.dtype != torch.float32 or t.shape != shape or not t.is_contiguous() or
                                      t.get_device() != self._sampler.device):
                    raise ValueError(f"out's scale and row_sum must be contiguous float32 {shape} on the sampler's device")
        if not self._sampler.handle:
            raise ValueError("the sampler is closed")
        a = _lib.pack_args(
            _RMS_NORM_ARGS, x.data_ptr(), residual.data_ptr() if residual is not None else 0, self._weight_ptr,
            out.residual.data_ptr() if out.residual is not None else 0, out.out.data_ptr(),
            out.scale.data_ptr() if out.scale is not None else 0, out.row_sum.data_ptr() if out.row_sum is not None else 0,
            rows, hidden, ld_x, ld_r, ld_ro, ld_out, dtype, *self._tail)
        st = self._L.gs_rms_norm(self._sampler.handle, a, _lib.current_stream(self._device) if stream is None else stream)
        if st != _lib.GS_OK:
            msg = self._sampler.last_error()
            raise ValueError(msg) if st == _lib.GS_EINVAL else SamplerError(st, msg)
        return out
