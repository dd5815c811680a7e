"""Microscaled 4-bit quantisation on the sm_100a library.

``quantize_fp4(x2, fmt)`` turns a matrix into an :class:`FP4Tensor`: E2M1 codes, a scale for
each block of a row, and for ``"nv"`` one power of two per row:

  ``"nv"``  blocks of 16, E4M3 scales amax / (6 r), r the row's power of two
  ``"mx"``  blocks of 32, E8M0 scales 2^(floor(log2 amax) - 2)

``fp4_mm`` (fp4_linear.py) multiplies such matrices on the block-scaled tensor cores, which
read the scales in the tiled order kept here.  The reference has no 4-bit operators: its
narrowest type is FP8 (fp8_quant.py:13-55).  Inference only, like the rest of the pack.
"""
from __future__ import annotations

import torch

from . import _lib

FP4_MAX = 6.0

_FMTS = {"nv": _lib.FVB_FP4_NV, "mx": _lib.FVB_FP4_MX}
_BLOCK = {"nv": 16, "mx": 32}
_DTYPES = {torch.bfloat16: _lib.FVB_BF16, torch.float16: _lib.FVB_F16, torch.float32: _lib.FVB_F32}


def fp4_format(fmt: str) -> int:
    try:
        return _FMTS[fmt]
    except KeyError:
        raise ValueError(f"unknown FP4 format {fmt!r} (nv|mx)") from None


def _dtype_code(dtype, name):
    try:
        return _DTYPES[dtype]
    except KeyError:
        raise ValueError(f"{name}: expected bf16, fp16 or fp32, got {dtype}") from None


class FP4Tensor:
    """A matrix [M, K] in microscaled 4-bit form.

    codes      uint8 [M, ceil(K / 32) * 16]: two codes to a byte, even element in the low
               nibble, zero codes past K
    scales     uint8, 512-byte tiles [ceil(M / 128), ceil(blocks / 4)]; block j of row m is
               byte (m % 32) * 16 + (m % 128) // 32 * 4 + j % 4 of tile (m // 128, j // 4)
    row_scale  fp32 [M] or [1] (``"nv"``; None = 1), None for ``"mx"``
    shape      (M, K);  fmt  "nv" or "mx"
    """

    __slots__ = ("shape", "fmt", "device", "_row_mode", "codes_ptr", "scales_ptr", "row_scale_ptr",
                 "_buf", "_codes", "_scales", "_row_scale")

    def __init__(self, codes, scales, row_scale, shape, fmt):
        code = fp4_format(fmt)
        M, K = shape
        pitch = (K + 31) // 32 * 16
        per = 4 * _BLOCK[fmt]
        tiles = (M + 127) // 128 * ((K + per - 1) // per)
        if codes.dtype != torch.uint8 or codes.numel() != M * pitch or not codes.is_contiguous():
            raise ValueError(f"FP4Tensor: codes must be contiguous uint8 [{M}, {pitch}], got "
                             f"{codes.dtype} {tuple(codes.shape)}")
        if scales.dtype != torch.uint8 or scales.numel() != tiles * 512 or not scales.is_contiguous():
            raise ValueError(f"FP4Tensor: scales must be contiguous uint8 of {tiles * 512} bytes, "
                             f"got {scales.dtype} {tuple(scales.shape)}")
        device = codes.device
        rows = 0
        if code == _lib.FVB_FP4_MX:
            if row_scale is not None:
                raise ValueError("FP4Tensor: mx has no row_scale")
        elif row_scale is not None:
            rows = row_scale.numel()
            if row_scale.dtype != torch.float32 or rows not in (1, M) \
                    or not row_scale.is_contiguous():
                raise ValueError("FP4Tensor: row_scale must be contiguous fp32 with 1 or M entries")
            if row_scale.device != device:
                raise ValueError("FP4Tensor: codes, scales and row_scale must be on one device")
        if scales.device != device:
            raise ValueError("FP4Tensor: codes, scales and row_scale must be on one device")
        self._codes, self._scales, self._row_scale, self._buf = codes, scales, row_scale, None
        self.codes_ptr, self.scales_ptr = codes.data_ptr(), scales.data_ptr()
        self.row_scale_ptr = None if row_scale is None else row_scale.data_ptr()
        self._row_mode = _lib.FVB_SCALE_ROW if rows and rows == M else _lib.FVB_SCALE_TENSOR
        self.shape = (M, K)
        self.fmt = fmt
        self.device = device

    # the buffers of a tensor the library made lie in one allocation and become tensors when
    # they are asked for
    @property
    def codes(self):
        if self._codes is None:
            M, K = self.shape
            pitch = (K + 31) // 32 * 16
            self._codes = self._buf[:M * pitch].view(M, pitch)
        return self._codes

    @property
    def scales(self):
        if self._scales is None:
            a = self.scales_ptr - self._buf.data_ptr()
            per = 4 * _BLOCK[self.fmt]
            n = (self.shape[0] + 127) // 128 * ((self.shape[1] + per - 1) // per) * 512
            self._scales = self._buf[a:a + n]
        return self._scales

    @property
    def row_scale(self):
        if self._row_scale is None and self._buf is not None and self.fmt == "nv":
            a = self.row_scale_ptr - self._buf.data_ptr()
            self._row_scale = self._buf[a:a + 4 * self.shape[0]].view(torch.float32)
        return self._row_scale

    def row_mode(self) -> int:
        """FVB_SCALE_ROW for one row scale a row, else FVB_SCALE_TENSOR."""
        return self._row_mode

    def __repr__(self):
        return f"FP4Tensor({self.fmt}, shape={self.shape}, device={self.device})"


def _empty(M: int, K: int, fmt: str, device) -> FP4Tensor:
    """An FP4Tensor of uninitialised buffers in one allocation (three cost 5 us more)."""
    t = FP4Tensor.__new__(FP4Tensor)
    per = 4 * _BLOCK[fmt]
    scales = (M * ((K + 31) // 32 * 16) + 511) // 512 * 512
    rows = scales + (M + 127) // 128 * ((K + per - 1) // per) * 512
    nv = fmt == "nv"
    buf = torch.empty(rows + 4 * M if nv else rows, dtype=torch.uint8, device=device)
    base = buf.data_ptr()
    t._buf, t._codes, t._scales, t._row_scale = buf, None, None, None
    t.codes_ptr, t.scales_ptr = base, base + scales
    t.row_scale_ptr = base + rows if nv else None
    t._row_mode = _lib.FVB_SCALE_ROW if nv and M else _lib.FVB_SCALE_TENSOR
    t.shape = (M, K)
    t.fmt = fmt
    t.device = buf.device
    return t


def require_cuda(q: FP4Tensor):
    if q.device.type != "cuda":
        _lib.require_cuda(q.codes)


def quantize_fp4(x2: torch.Tensor, fmt: str = "nv") -> FP4Tensor:
    """x2 [M, K] bf16, fp16 or fp32 (unit column stride, any row stride) -> FP4Tensor.

    code = e2m1(x / scale), to nearest, ties to even, saturating at 6.  A block with a NaN or
    an infinity gets a NaN scale; the row's power of two comes from its finite values.
    """
    code = fp4_format(fmt)
    _lib.require_cuda(x2)
    if x2.dim() != 2:
        raise ValueError(f"quantize_fp4: expected a 2-D [M, K] tensor, got {tuple(x2.shape)}")
    dt = _dtype_code(x2.dtype, "quantize_fp4")
    M, K = x2.shape
    if (K > 1 and x2.stride(1) != 1) or (M > 1 and x2.stride(0) < K):
        x2 = x2.contiguous()
    q = _empty(M, K, fmt, x2.device)
    _lib.call("fvb_quant_fp4", x2.data_ptr(), dt, x2.stride(0) if M > 1 else K, M, K, code,
              q.codes_ptr, q.scales_ptr, q.row_scale_ptr, _lib.stream_of(x2))
    return q


def dequantize_fp4(q: FP4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values an FP4Tensor stands for, [M, K]; one rounding to `dtype` (none for codes of
    quantize_fp4 in bf16 or fp32: they hold a code times a scale exactly)."""
    require_cuda(q)
    dt = _dtype_code(dtype, "dequantize_fp4")
    M, K = q.shape
    out = torch.empty((M, K), dtype=dtype, device=q.device)
    _lib.call("fvb_dequant_fp4", q.codes_ptr, q.scales_ptr, q.row_scale_ptr, q._row_mode, M, K,
              _FMTS[q.fmt], dt, out.data_ptr(), _lib.stream_of(out))
    return out
