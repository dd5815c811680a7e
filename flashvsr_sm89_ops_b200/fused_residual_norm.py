"""The seam between two branches of a block with norms on both sides of a branch, in one pass.

``fused_residual_norm`` adds a branch's output to the residual stream, after an optional norm
and gate and with a scale on the stream, and norms and modulates the result for the next
branch, in bf16 and / or as the 4-bit codes that fp4_mm and ffn_fp4 take.  The wider form of
gate_add_ln_modulate / gate_add_layer_norm (fused_adaln.py): those reproduce the reference's
bf16 chain bit for bit, this one stays in fp32 between its loads and stores.
"""
from __future__ import annotations

import torch

from . import _lib
from .fp4_quant import _empty, fp4_format

_NORMS = {None: _lib.FVB_NORM_NONE, "rms": _lib.FVB_NORM_RMS, "layer": _lib.FVB_NORM_LAYER}


def _operand(t, n, what, device, items=0):
    """t of n entries as the kernel takes it.  items: t has a row for each of so many batch items; a
    3-D t of another shape, [1, L, D] with L = items say, would mean something else."""
    if t is None:
        return None
    if items > 1 and t.dim() == 3:
        if t.shape != (items, 1, n // items):
            raise ValueError(f"fused_residual_norm: {what} must be [{items}, 1, {n // items}], got {tuple(t.shape)}")
    elif t.numel() != n:
        raise ValueError(f"fused_residual_norm: {what} must have {n} entries, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"fused_residual_norm: {what} is on {t.device}, x on {device}")
    if t.dtype != torch.bfloat16:
        t = t.to(torch.bfloat16)
    return t if t.is_contiguous() else t.contiguous()


def fused_residual_norm(x: torch.Tensor, y: torch.Tensor, *, gate: torch.Tensor | None = None,
                        residual_scale: float = 1.0, post_norm: str | None = None,
                        post_weight: torch.Tensor | None = None,
                        post_bias: torch.Tensor | None = None, post_eps: float | None = None,
                        norm: str = "layer", weight: torch.Tensor | None = None,
                        bias: torch.Tensor | None = None, scale: torch.Tensor | None = None,
                        shift: torch.Tensor | None = None, eps: float = 1e-6,
                        emit_fp4: str | None = None, want_out: bool = True):
    """x_new = residual_scale * x + gate * (post_norm(y) * post_weight + post_bias)
       h     = (norm(x_new) * weight + bias) * (1 + scale) + shift

    x, y [B, L, D] bf16.  post_norm None, "rms" or "layer"; norm "rms" or "layer".  gate
    [B, 1, D] or [B, L, D]; scale and shift [B, 1, D]; the weights and biases [D]; any of them
    None.  Returns (x_new, h), or with emit_fp4 ("nv" or "mx") (x_new, h, FP4Tensor [B * L, D]
    of the unrounded h); h is None when want_out=False.  D a multiple of 8, at most 16384.
    """
    _lib.require_cuda(x, y)
    if x.dim() != 3:
        raise ValueError(f"fused_residual_norm: expected x [B, L, D], got {tuple(x.shape)}")
    if x.dtype != torch.bfloat16 or y.dtype != torch.bfloat16:
        raise ValueError(f"fused_residual_norm: expected bf16, got {x.dtype} and {y.dtype}")
    if y.shape != x.shape:
        raise ValueError(f"fused_residual_norm: y {tuple(y.shape)} does not match x {tuple(x.shape)}")
    if post_norm not in _NORMS or norm not in ("rms", "layer"):
        raise ValueError(f"fused_residual_norm: norms are 'rms' or 'layer', got {post_norm!r}, {norm!r}")
    if post_norm is None and (post_weight is not None or post_bias is not None):
        raise ValueError("fused_residual_norm: post_weight / post_bias without a post_norm")
    fmt = 0 if emit_fp4 is None else fp4_format(emit_fp4)
    if not want_out and not fmt:
        raise ValueError("fused_residual_norm: want_out=False needs emit_fp4")
    B, L, D = x.shape
    dev = x.device
    if y.device != dev:
        raise ValueError(f"fused_residual_norm: y is on {y.device}, x on {dev}")
    x = x if x.is_contiguous() else x.contiguous()
    y = y if y.is_contiguous() else y.contiguous()
    gate_rows = 0
    if gate is not None:
        if L > 1 and gate.numel() == B * L * D and (gate.dim() != 3 or gate.shape == x.shape):
            gate_rows = 1
            gate = _operand(gate, B * L * D, "gate", dev)
        else:
            gate = _operand(gate, B * D, "gate", dev, B)
    scale = _operand(scale, B * D, "scale", dev, B)
    shift = _operand(shift, B * D, "shift", dev, B)
    post_weight = _operand(post_weight, D, "post_weight", dev)
    post_bias = _operand(post_bias, D, "post_bias", dev)
    weight = _operand(weight, D, "weight", dev)
    bias = _operand(bias, D, "bias", dev)
    # NULL (0) for what is absent; the kernel reads 16-byte vectors
    xp, yp = x.data_ptr(), y.data_ptr()
    gp = gate.data_ptr() if gate is not None else 0
    pwp = post_weight.data_ptr() if post_weight is not None else 0
    pbp = post_bias.data_ptr() if post_bias is not None else 0
    wp = weight.data_ptr() if weight is not None else 0
    bp = bias.data_ptr() if bias is not None else 0
    scp = scale.data_ptr() if scale is not None else 0
    shp = shift.data_ptr() if shift is not None else 0
    if (xp | yp | gp | pwp | pbp | wp | bp | scp | shp) & 15:
        copies = [t.clone() if t is not None and t.data_ptr() & 15 else t
                  for t in (x, y, gate, post_weight, post_bias, weight, bias, scale, shift)]
        xp, yp, gp, pwp, pbp, wp, bp, scp, shp = (0 if t is None else t.data_ptr() for t in copies)
    x_new = torch.empty_like(x)
    h = torch.empty_like(x) if want_out else None
    q = _empty(B * L, D, emit_fp4, dev) if fmt else None
    _lib.call("fvb_residual_norm", xp, yp, gp, gate_rows, float(residual_scale), _NORMS[post_norm],
              pwp, pbp, float(eps if post_eps is None else post_eps), _NORMS[norm], wp, bp, scp, shp,
              float(eps), B, L, D, x_new.data_ptr(), h.data_ptr() if want_out else 0, fmt,
              q.codes_ptr if fmt else None, q.scales_ptr if fmt else None,
              q.row_scale_ptr if fmt else None, _lib.stream_of(x))
    return (x_new, h, q) if fmt else (x_new, h)
