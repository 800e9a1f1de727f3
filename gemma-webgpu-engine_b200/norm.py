"""Residual + RMS norm with an 8-bit output (gs_rms_norm): the pass before a product.

Per row, in float32: h = x + residual, y = h · (mean(h²) + eps)^-1/2 · (weight_offset + weight);
h is kept for the next layer, y goes out as float32 / bfloat16, as e4m3 codes with a float32
scale per row or per group of columns, or (``srq_scale``) on the int8 grid that
``GpuLmHead`` reads, with its row sum.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

from . import _lib
from .sampling import SamplerError


@dataclass
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
        a = _lib.GsRmsNormArgs()
        if weight is not None:
            a.weight = weight.data_ptr()
            a.weight_dtype = _lib.GS_DTYPE_BF16 if weight.dtype == torch.bfloat16 else _lib.GS_DTYPE_F32
        a.hidden = self.hidden
        a.out_dtype = {"bf16": _lib.GS_DTYPE_BF16, "f32": _lib.GS_DTYPE_F32, "e4m3": _lib.GS_DTYPE_E4M3,
                       "srq": _lib.GS_DTYPE_F32}[out]
        a.group = self.group
        a.eps, a.weight_offset, a.srq_scale = float(eps), float(weight_offset), float(srq_scale)
        self._fixed = bytes(a)

    def _rows(self, t, what, like=None):
        if t.dim() != 2 or t.shape[1] != self.hidden:
            raise ValueError(f"{what} must be [rows, {self.hidden}]")
        if t.stride(1) != 1 and self.hidden > 1:
            raise ValueError(f"{what} rows must be contiguous")
        if t.device != self._device:
            raise ValueError(f"{what} must be on the sampler's device")
        if like is not None and (t.dtype != like.dtype or t.shape[0] != like.shape[0]):
            raise ValueError(f"{what} must have x's type and rows")
        return t.stride(0) if t.shape[0] > 1 else self.hidden

    def __call__(self, x, residual=None, *, out: RmsNormResult | None = None, stream=None) -> RmsNormResult:
        """The norm of x (+ residual), both [rows, hidden] float32 or bfloat16.  ``out``: a result
        to write into (its ``residual`` may be the residual itself)."""
        torch = self._torch
        if x.dtype == torch.bfloat16:
            dtype = _lib.GS_DTYPE_BF16
        elif x.dtype == torch.float32:
            dtype = _lib.GS_DTYPE_F32
        else:
            raise ValueError("x must be float32 or bfloat16")
        a = _lib.GsRmsNormArgs.from_buffer_copy(self._fixed)
        a.ld_x = self._rows(x, "x")
        rows = x.shape[0]
        a.dtype, a.rows, a.x = dtype, rows, x.data_ptr()
        if residual is not None:
            a.ld_residual = self._rows(residual, "residual", x)
            a.residual = residual.data_ptr()
        if out is None:
            dev = self._device
            out = RmsNormResult(
                torch.empty((rows, self.hidden), dtype=self._out_type, device=dev),
                torch.empty((rows, self.groups), dtype=torch.float32, device=dev) if self.out == "e4m3" else None,
                torch.empty((rows, self.hidden), dtype=x.dtype, device=dev) if residual is not None else None,
                torch.empty(rows, dtype=torch.float32, device=dev) if self.out == "srq" else None)
            a.ld_out = a.ld_residual_out = self.hidden
        else:
            a.ld_out = self._rows(out.out, "out.out")
            if out.out.dtype != self._out_type or out.out.shape[0] != rows:
                raise ValueError("out.out must have the output type and x's rows")
            if out.residual is not None:
                a.ld_residual_out = self._rows(out.residual, "out.residual", x)
            for t, shape in ((out.scale, (rows, self.groups)), (out.row_sum, (rows,))):
                if t is not None and (t.dtype != torch.float32 or tuple(t.shape) != shape or not t.is_contiguous()):
                    raise ValueError(f"out's scale and row_sum must be contiguous float32 {shape}")
        a.out = out.out.data_ptr()
        if out.residual is not None:
            a.residual_out = out.residual.data_ptr()
        if out.scale is not None:
            a.out_scale = out.scale.data_ptr()
        if out.row_sum is not None:
            a.row_sum = out.row_sum.data_ptr()
        if stream is None:
            stream = _lib.current_stream(self._device)
        st = self._L.gs_rms_norm(self._sampler.handle, ctypes.byref(a), stream)
        if st != _lib.GS_OK:
            msg = self._sampler.last_error()
            raise ValueError(msg) if st == _lib.GS_EINVAL else SamplerError(st, msg)
        return out
