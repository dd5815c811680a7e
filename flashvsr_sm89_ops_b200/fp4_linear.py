"""4-bit Linear and FFN on hand-written block-scaled tcgen05 products (sm_100a).

The 4-bit counterparts of fp8_linear.py and fp8_ffn.py (whose reference is
fp8_linear.py:16-67 and fp8_ffn.py:75-115): the weight is quantised once, every forward
quantises its input and multiplies.  ``FP4FFN`` keeps its hidden state in 4 bits: the first
product's epilogue applies bias and GELU(tanh) and writes mx codes, so no 16-bit hidden state
exists.  Inference only, like the rest of the pack.
"""
from __future__ import annotations

import re

import torch
import torch.nn as nn

from . import _lib
from .fp4_quant import _FMTS, FP4Tensor, fp4_format, quantize_fp4, require_cuda
from .fp8_linear import FP8Linear


def _vector(t, n, what, device):
    """A bf16 vector of n entries for the kernel (None stays None)."""
    if t is None:
        return None
    if t.dtype is torch.bfloat16 and t.shape == (n,) and t.device == device and t.is_contiguous():
        return t
    if t.numel() != n:
        raise ValueError(f"{what} must have {n} entries, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, the operands on {device}")
    if t.dtype != torch.bfloat16:
        t = t.to(torch.bfloat16)
    return t.reshape(-1).contiguous() if t.dim() != 1 or not t.is_contiguous() else t


def _residual(r, M, N, what, device):
    """(residual as [M, N] with unit column stride, its row pitch)."""
    if r is None:
        return None, 0
    if r.dtype is torch.bfloat16 and r.shape == (M, N) and r.device == device and r.is_contiguous():
        return r, N
    if r.dtype != torch.bfloat16 or r.numel() != M * N or r.shape[-1] != N:
        raise ValueError(f"{what}: residual must be bf16 [{M}, {N}], got {r.dtype} {tuple(r.shape)}")
    if r.device != device:
        raise ValueError(f"{what}: residual is on {r.device}, the operands on {device}")
    if r.dim() != 2:
        r = r.reshape(M, N)
    if (N > 1 and r.stride(1) != 1) or (M > 1 and r.stride(0) < N):
        r = r.contiguous()
    return r, (r.stride(0) if M > 1 else N)


def _out(out, M, N, what, device):
    if out is None:
        return torch.empty((M, N), dtype=torch.bfloat16, device=device)
    if out.dtype != torch.bfloat16 or out.numel() != M * N or not out.is_contiguous() \
            or out.device != device:
        raise ValueError(f"{what}: out must be a contiguous bf16 [{M}, {N}] tensor on {device}")
    return out


def fp4_mm(a: FP4Tensor, w: FP4Tensor, bias: torch.Tensor | None = None,
           out: torch.Tensor | None = None, residual: torch.Tensor | None = None,
           gate: torch.Tensor | None = None) -> torch.Tensor:
    """bf16(a w^T + bias), or bf16(residual + gate * (a w^T + bias)) with a residual.

    a [M, K] and w [N, K] of the same format; bias and gate [N], residual [M, N].  fp32 sums
    and epilogue, one rounding.  out (contiguous [M, N]) may be the residual.
    """
    require_cuda(a)
    M, K = a.shape
    N = w.shape[0]
    dev = a.device
    if a.fmt != w.fmt:
        raise ValueError(f"fp4_mm: formats differ ({a.fmt} x {w.fmt})")
    if w.shape[1] != K:
        raise ValueError(f"fp4_mm: K mismatch {a.shape} x {w.shape}")
    if w.device != dev:
        raise ValueError("fp4_mm: operands are on different devices")
    if gate is not None and residual is None:
        raise ValueError("fp4_mm: gate needs a residual")
    bias = _vector(bias, N, "fp4_mm: bias", dev)
    gate = _vector(gate, N, "fp4_mm: gate", dev)
    residual, ldr = _residual(residual, M, N, "fp4_mm", dev)
    out = _out(out, M, N, "fp4_mm", dev)
    ptr = _lib.ptr
    _lib.call("fvb_fp4_gemm", a.codes_ptr, a.scales_ptr, a.row_scale_ptr, a._row_mode, w.codes_ptr,
              w.scales_ptr, w.row_scale_ptr, w._row_mode, _FMTS[a.fmt], ptr(bias), ptr(residual),
              ldr, ptr(gate), M, N, K, out.data_ptr(), _lib.stream_of(out))
    return out


def ffn_fp4(a: FP4Tensor, w0: FP4Tensor, b0: torch.Tensor | None, w2: FP4Tensor,
            b2: torch.Tensor | None, residual: torch.Tensor | None = None,
            gate: torch.Tensor | None = None, out: torch.Tensor | None = None,
            workspace: torch.Tensor | None = None) -> torch.Tensor:
    """y = mx(gelu_tanh(a w0^T + b0)) w2^T + b2 in one call; bf16(y), or
    bf16(residual + gate * y) with a residual.

    a [M, D] and w0 [F, D] share a format, w2 [N, F] is mx (the hidden state's format: its
    blocks need nothing of the rest of their row, so the first product writes them itself).
    workspace: uint8, at least fvb_fp4_ffn_workspace_bytes(M, F), 256-byte aligned.
    """
    require_cuda(a)
    M, D = a.shape
    F, N = w0.shape[0], w2.shape[0]
    dev = a.device
    if a.fmt != w0.fmt:
        raise ValueError(f"ffn_fp4: formats differ ({a.fmt} x {w0.fmt})")
    if w2.fmt != "mx":
        raise ValueError("ffn_fp4: w2 must be mx, the hidden state's format")
    if w0.shape[1] != D or w2.shape[1] != F:
        raise ValueError(f"ffn_fp4: shapes {a.shape}, {w0.shape}, {w2.shape} do not chain")
    if w0.device != dev or w2.device != dev:
        raise ValueError("ffn_fp4: operands are on different devices")
    if gate is not None and residual is None:
        raise ValueError("ffn_fp4: gate needs a residual")
    b0 = _vector(b0, F, "ffn_fp4: b0", dev)
    b2 = _vector(b2, N, "ffn_fp4: b2", dev)
    gate = _vector(gate, N, "ffn_fp4: gate", dev)
    residual, ldr = _residual(residual, M, N, "ffn_fp4", dev)
    out = _out(out, M, N, "ffn_fp4", dev)
    need = _lib.load().fvb_fp4_ffn_workspace_bytes(M, F)
    if workspace is None:
        workspace = torch.empty(max(need, 256), dtype=torch.uint8, device=dev)
    elif workspace.numel() * workspace.element_size() < need or workspace.device != dev \
            or not workspace.is_contiguous():
        raise ValueError(f"ffn_fp4: workspace needs {need} contiguous bytes on {dev}")
    ptr = _lib.ptr
    _lib.call("fvb_fp4_ffn", a.codes_ptr, a.scales_ptr, a.row_scale_ptr, a._row_mode, w0.codes_ptr,
              w0.scales_ptr, w0.row_scale_ptr, w0._row_mode, _FMTS[a.fmt], ptr(b0), w2.codes_ptr,
              w2.scales_ptr, ptr(b2), ptr(residual), ldr, ptr(gate), M, D, F, N, out.data_ptr(),
              workspace.data_ptr(), _lib.stream_of(out))
    return out


def _quantize_weight(w: torch.Tensor, fmt: str):
    """(codes, scales, row scale) of a weight, in buffers of their own on the weight's device.  A
    weight on the host (a model that is moved to the GPU after its conversion) goes through the
    current CUDA device, since the quantiser has no other form."""
    if not w.is_cuda and not torch.cuda.is_available():
        raise ValueError("FP4Linear: quantising a weight takes a CUDA device (sm_100a)")
    q = quantize_fp4(w if w.is_cuda else w.cuda(), fmt)
    parts = (q.codes, q.scales, q.row_scale)
    return tuple(None if t is None else t.clone() if w.is_cuda else t.to(w.device) for t in parts)


class FP4Linear(nn.Module):
    """nn.Linear replacement with 4-bit weights and activations (cf. FP8Linear).  The weight is
    quantised once, here; a linear on the host stays there."""

    def __init__(self, linear: nn.Linear, fmt: str = "nv"):
        super().__init__()
        fp4_format(fmt)
        self.fmt = fmt
        self.in_features = linear.in_features
        self.out_features = linear.out_features
        codes, scales, row_scale = _quantize_weight(linear.weight.detach(), fmt)
        self.weight = nn.Parameter(codes, requires_grad=False)
        self.register_buffer("w_scales", scales, persistent=False)
        # the fp32 row scales' bits as integers: a cast of the whole model, to fp16 say, where 2^-25
        # is 0, leaves them alone
        bits = None if row_scale is None else row_scale.view(torch.int32)
        self.register_buffer("w_row_scale_bits", bits, persistent=False)
        if linear.bias is not None:
            self.bias = nn.Parameter(linear.bias.detach().to(torch.bfloat16).clone(),
                                     requires_grad=False)
        else:
            self.bias = None

    def weight_fp4(self) -> FP4Tensor:
        bits = self.w_row_scale_bits
        return FP4Tensor(self.weight.data, self.w_scales,
                         None if bits is None else bits.view(torch.float32),
                         (self.out_features, self.in_features), self.fmt)

    def forward(self, x):
        shape = x.shape
        y = fp4_mm(quantize_fp4(x.reshape(-1, shape[-1]), self.fmt), self.weight_fp4(), self.bias)
        return y.reshape(*shape[:-1], self.out_features)

    def extra_repr(self):
        return f"in={self.in_features}, out={self.out_features}, fmt={self.fmt}"


class FP4FFN(nn.Module):
    """Replacement for a DiT FFN ``Sequential(Linear, GELU(tanh), Linear)`` whose two Linears
    are FP4Linear, the second mx (cf. FP8FFN)."""

    def __init__(self, lin0: FP4Linear, lin2: FP4Linear):
        super().__init__()
        if lin2.fmt != "mx":
            raise ValueError("FP4FFN: the second linear must be mx")
        self.lin0 = lin0
        self.lin2 = lin2

    def ffn(self, a: FP4Tensor, residual=None, gate=None):
        """The FFN of an already quantised input, with the block's gated residual."""
        return ffn_fp4(a, self.lin0.weight_fp4(), self.lin0.bias, self.lin2.weight_fp4(),
                       self.lin2.bias, residual=residual, gate=gate)

    def forward(self, x):
        shape = x.shape
        y = self.ffn(quantize_fp4(x.reshape(-1, shape[-1]), self.lin0.fmt))
        return y.reshape(*shape[:-1], self.lin2.out_features)


_PATTERNS = {"self": r"^blocks\.\d+\.self_attn\.[qkvo]$", "cross": r"^blocks\.\d+\.cross_attn\.[qkvo]$"}


def convert_linears_fp4(model: nn.Module, parts=("ffn",), fmt: str = "nv") -> int:
    """Swap the DiT blocks' Linears of `parts` (ffn, self, cross) for 4-bit ones; returns the
    count.  ``blocks.i.ffn`` becomes an FP4FFN whose first linear has `fmt`.  Same module names
    as convert_linears_fp8 (fp8_linear.py:45-67).  What is 4-bit in `fmt` already stays; a part
    that was converted to FP8 or to the other format, its full-precision weights gone, is refused
    before anything is converted."""
    fp4_format(fmt)
    unknown = set(parts) - {"ffn", "self", "cross"}
    if unknown:
        raise ValueError(f"convert_linears_fp4: unknown parts {sorted(unknown)} (ffn|self|cross)")
    pats = [re.compile(_PATTERNS[p]) for p in parts if p in _PATTERNS]
    ffn = re.compile(r"^blocks\.\d+\.ffn$") if "ffn" in parts else None
    todo = []
    for name, mod in list(model.named_modules()):
        is_ffn = ffn is not None and ffn.match(name)
        if not is_ffn and not any(p.match(name) for p in pats):
            continue
        # the linear that an FFN, of whichever kind, begins with speaks for it
        lin = mod if not is_ffn else mod[0] if isinstance(mod, nn.Sequential) else getattr(mod, "lin0", None)
        if isinstance(lin, FP8Linear) or (isinstance(lin, FP4Linear) and lin.fmt != fmt):
            kind = "FP8" if isinstance(lin, FP8Linear) else lin.fmt
            raise ValueError(f"convert_linears_fp4: {name} is already {kind}, it cannot become {fmt}")
        if type(lin) is nn.Linear and (not is_ffn or type(mod[2]) is nn.Linear):
            todo.append((name, mod, is_ffn))
    n = 0
    for name, mod, is_ffn in todo:
        parent_name, _, leaf = name.rpartition(".")
        new = FP4FFN(FP4Linear(mod[0], fmt), FP4Linear(mod[2], "mx")) if is_ffn else FP4Linear(mod, fmt)
        setattr(model.get_submodule(parent_name) if parent_name else model, leaf, new)
        n += 2 if is_ffn else 1
    return n
