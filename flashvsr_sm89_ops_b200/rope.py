"""Rotary positions of q and k in one launch on the sm_100a library.

``fused_rope(q, k, positions, rope)`` is the general form beside fused_rms_rope (which takes a
table of complex numbers, interleaved pairs and whole heads, after its norm): a :class:`Rope`
holds the frequencies, and the angles are formed in the kernel from integer positions.  The
gradient is the inverse rotation; autograd takes it, and ``inverse=True`` is it.
"""
from __future__ import annotations

import math

import torch
import torch.autograd.forward_ad as forward_ad

from . import _lib
from .fp4_quant import _dtype_code

_POS64 = {torch.int32: 0, torch.int64: 1}
_SCALINGS = (None, "linear", "ntk", "yarn")


def _frequencies(d: int, theta: float, scaling, factor: float, original_len, beta_fast: float, beta_slow: float):
    """Angles a position, of the d / 2 pairs of one axis."""
    if scaling == "ntk" and d > 2:
        theta = theta * factor ** (d / (d - 2))
    w = [theta ** (-2 * i / d) for i in range(d // 2)]
    if scaling == "linear":
        w = [x / factor for x in w]
    elif scaling == "yarn":
        # pairs that turn more than beta_fast times over the original length keep their
        # frequency, those below beta_slow turns are stretched by the factor, a ramp between
        def pair(turns):
            return d * math.log(original_len / (turns * 2 * math.pi)) / (2 * math.log(theta))

        # (published as clipped to the channels, not to the pairs: the ramp may end behind the last pair)
        low, high = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), d - 1)
        ramp = [min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(d // 2)]
        w = [x * (1 - r) + x / factor * r for x, r in zip(w, ramp)]
    return w


class Rope:
    """Frequencies of a rotary embedding of the first `rotary_dim` channels of a head.

    layout   "interleaved": pair i is channels (2i, 2i + 1); "half": (i, i + rotary_dim / 2)
    theta    base: pair i turns by theta^(-2 i / d) a position
    scaling  for contexts `factor` times longer than trained: None; "linear" (positions divided
             by the factor); "ntk" (theta times factor^(d / (d - 2))); "yarn" (by parts, between
             beta_fast and beta_slow turns over `original_len` positions, and the rotated channels
             multiplied by 0.1 ln(factor) + 1, or by attention_factor)
    axes     channels of each axis for positions of several coordinates, (44, 42, 42) for the
             frame, row and column of a 128-channel head; each axis has its own frequencies
    """

    def __init__(self, rotary_dim: int, *, theta: float = 10000.0, layout: str = "interleaved",
                 scaling: str | None = None, factor: float = 1.0, original_len: int | None = None,
                 beta_fast: float = 32.0, beta_slow: float = 1.0, attention_factor: float | None = None,
                 axes=None, device="cuda"):
        if rotary_dim < 0 or rotary_dim % 2:
            raise ValueError(f"Rope: rotary_dim must be even, got {rotary_dim}")
        if layout not in ("interleaved", "half"):
            raise ValueError(f"Rope: unknown layout {layout!r} (interleaved|half)")
        if scaling not in _SCALINGS:
            raise ValueError(f"Rope: unknown scaling {scaling!r} (linear|ntk|yarn)")
        if not theta > 1 or not math.isfinite(theta):
            raise ValueError(f"Rope: theta must be above 1, got {theta}")
        if scaling is not None and not (factor >= 1 and math.isfinite(factor)):
            raise ValueError(f"Rope: factor must be at least 1, got {factor}")
        if scaling == "yarn" and (not original_len or original_len < 1 or not 0 < beta_slow < beta_fast):
            raise ValueError("Rope: yarn needs original_len and 0 < beta_slow < beta_fast")
        dims = (rotary_dim,) if axes is None else tuple(int(d) for d in axes)
        if not 1 <= len(dims) <= 16 or any(d < 0 or d % 2 for d in dims) or sum(dims) != rotary_dim:
            raise ValueError(f"Rope: axes must be up to 16 even counts that add up to {rotary_dim}, got {dims}")
        w = [x for d in dims for x in _frequencies(d, theta, scaling, factor, original_len, beta_fast, beta_slow)]
        # turns a position as a fraction of 2^64
        turns = [round(x / (2 * math.pi) * 2.0 ** 64) for x in w]
        self.rotary_dim, self.layout, self.axes = rotary_dim, layout, len(dims)
        self.half = layout == "half"
        self.scale = 1.0
        if scaling == "yarn":
            self.scale = 0.1 * math.log(factor) + 1 if attention_factor is None else float(attention_factor)
        self._tensors = (torch.tensor(turns, dtype=torch.int64, device=device),
                         torch.tensor([a for a, d in enumerate(dims) for _ in range(d // 2)], dtype=torch.int32,
                                      device=device))
        self._bind()

    def _bind(self):
        self.device = self.freq.device
        self.index = self.freq.get_device()  # -1 on the host
        self._freq, self._axis = self.freq.data_ptr(), self.axis.data_ptr()

    # a copy (of a model that holds one, say) has tensors, and so addresses, of its own
    def __setstate__(self, state):
        self.__dict__.update(state)
        self._bind()

    # the calls hold the addresses of these
    freq = property(lambda self: self._tensors[0])
    axis = property(lambda self: self._tensors[1])

    def __repr__(self):
        return f"Rope({self.rotary_dim}, layout={self.layout!r}, axes={self.axes}, scale={self.scale})"


def _rows(x, what, name):
    """x [T, H, D] or [B, L, H, D] as rows with unit stride inside a head: (x, T, H, D, its strides of
    tokens and heads)."""
    s, n = x.stride(), x.shape
    if len(n) == 3 and (s[2] == 1 or n[2] < 2):
        return x, n[0], n[1], n[2], s[0], s[1]
    if len(n) == 4:
        x = x.flatten(0, 1) if s[0] == n[1] * s[1] else x.contiguous().flatten(0, 1)
    if x.dim() != 3:
        raise ValueError(f"{name}: {what} must be [T, H, D] or [B, L, H, D], got {tuple(x.shape)}")
    if x.shape[2] > 1 and x.stride(2) != 1:
        x = x.contiguous()
    return x, *x.shape, x.stride(0), x.stride(1)


def _positions(positions, rope, T, index, name):
    if positions.get_device() != index:
        raise ValueError(f"{name}: positions are on {positions.device}, q on cuda:{index}")
    if positions.dtype not in _POS64:
        raise ValueError(f"{name}: positions must be int32 or int64, got {positions.dtype}")
    if positions.numel() != T * rope.axes or (rope.axes > 1 and positions.shape[-1] != rope.axes):
        raise ValueError(f"{name}: positions must be one of {rope.axes} coordinate(s) for each of {T} tokens, "
                         f"got {tuple(positions.shape)}")
    return positions if positions.is_contiguous() else positions.contiguous()


def _out(out, x, what, name):
    """The tensor that x's rotation goes to, and its rows' strides of tokens and heads."""
    if out is None:
        n = x.shape
        return torch.empty_like(x, memory_format=torch.contiguous_format), n[-2] * n[-1], n[-1]
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError(f"{name}: {what} must be {x.dtype} {tuple(x.shape)} on {x.device}")
    s = out.stride()
    if len(s) == 4 and s[0] != out.shape[1] * s[1] and out.shape[0] > 1:
        raise ValueError(f"{name}: the items of {what} must follow each other")
    if s[-1] != 1 and out.shape[-1] > 1:
        raise ValueError(f"{name}: {what} must have unit stride inside a head")
    return out, s[-3], s[-2]


def _clash(a, b, D):
    """Whether two sets of rows share an element.  Each: address, T, H, strides of tokens and heads, bytes an
    element; rows of D elements.  Sets of different strides that reach into each other count as such."""
    pa, Ta, Ha, ta, ha, e = a
    pb, Tb, Hb, tb, hb, _ = b
    if not Ta or not Tb or not Ha or not Hb:
        return False
    if pa + ((Ta - 1) * ta + (Ha - 1) * ha + D) * e <= pb or pb + ((Tb - 1) * tb + (Hb - 1) * hb + D) * e <= pa:
        return False
    t, h = (ta if Ta > 1 else tb), (ha if Ha > 1 else hb)  # the stride of an axis of one is any number
    if (Tb > 1 and t != tb) or (Hb > 1 and h != hb) or (pb - pa) % e:
        return True
    d = (pb - pa) // e
    if Ta == 1 and Tb == 1:
        t = 0
    elif t and (Ha - 1) * h + D <= d % t <= t - (Hb - 1) * h - D:
        return False  # beside each other in every token
    for i in range(1 - Ha, Hb):
        c = d + i * h
        at = (-c // t, -(c // t)) if t else (0,)
        if any(abs(c + min(max(n, 1 - Ta), Tb - 1) * t) < D for n in at):
            return True
    return False


def _own(rows, D, what, name):
    """Refuses an output whose rows lie over each other."""
    _, T, H, t, h, _ = rows
    (s0, n0), (s1, n1) = sorted(((t, T), (h, H))) if T > 1 and H > 1 else ((h, H), (t, T))
    inner = (n0 - 1) * s0 + D if n0 > 1 else D
    if T and H and ((n0 > 1 and s0 < D) or (n1 > 1 and s1 < inner)):
        raise ValueError(f"{name}: rows of {what} lie over each other")


def _apart(rows, others, D, what, name):
    """Refuses an output that shares elements with another tensor of the call: others are (rows, its
    name, whether being that very tensor is fine)."""
    _own(rows, D, what, name)
    for other, named, same in others:
        if same and rows[0] == other[0] and rows[1:3] == other[1:3] and \
                (rows[1] < 2 or rows[3] == other[3]) and (rows[2] < 2 or rows[4] == other[4]):
            continue
        if _clash(rows, other, D):
            raise ValueError(f"{name}: {what} lies over {named}")


def _run(q, k, positions, rope, inverse, out_q, out_k):
    name = "fused_rope"
    dt = _dtype_code(q.dtype, name)
    index = q.get_device()
    q3, T, Hq, D, st, sh = _rows(q, "q", name)
    if rope.rotary_dim > D:
        raise ValueError(f"{name}: rotary_dim {rope.rotary_dim} of a head of {D}")
    if rope.index != index:
        raise ValueError(f"{name}: the Rope is on {rope.device}, q on {q.device}")
    positions = _positions(positions, rope, T, index, name)
    oq, ot, oh = _out(out_q, q, "out_q", name)
    if k is None:
        if out_k is not None:
            raise ValueError(f"{name}: out_k without k")
        ok, kargs = None, (0, 0, 0, 0, 0, 0, 0)
    else:
        if k.dtype != q.dtype or k.get_device() != index:
            raise ValueError(f"{name}: k is {k.dtype} on {k.device}, q {q.dtype} on {q.device}")
        k3, Tk, Hk, Dk, kt, kh = _rows(k, "k", name)
        if Tk != T or Dk != D:
            raise ValueError(f"{name}: k {tuple(k.shape)} does not match q {tuple(q.shape)}")
        ok, kot, koh = _out(out_k, k, "out_k", name)
        kargs = (k3.data_ptr(), kt, kh, Hk, ok.data_ptr(), kot, koh)
    if out_q is not None or out_k is not None:
        e = q.element_size()
        ins = [((q3.data_ptr(), T, Hq, st, sh, e), "q")]
        if k is not None:
            ins.append(((k3.data_ptr(), T, Hk, kt, kh, e), "k"))
        rows = (oq.data_ptr(), T, Hq, ot, oh, e)
        if out_q is not None:
            _apart(rows, [(r, n, n == "q") for r, n in ins], D, "out_q", name)
        if out_k is not None:
            _apart((ok.data_ptr(), T, Hk, kot, koh, e), [(r, n, n == "k") for r, n in ins] + [(rows, "out_q", False)], D,
                   "out_k", name)
    _lib.call_on(index, "fvb_rope",
                 _lib.ROPE_ARGS(q3.data_ptr(), st, sh, Hq, oq.data_ptr(), ot, oh, *kargs, T, D, rope.rotary_dim,
                                rope.half, dt, positions.data_ptr(), _POS64[positions.dtype], rope.axes, rope._freq,
                                rope._axis, rope.scale, inverse), _lib.stream_of(q))
    return oq, ok


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, rope, inverse):
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)
        ctx.rope, ctx.inverse, ctx.two = rope, inverse, k is not None
        oq, ok = _run(q, k, positions, rope, inverse, None, None)
        return (oq, ok) if k is not None else oq

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk=None):
        positions, = ctx.saved_tensors
        if gk is None:
            return _run(gq, None, positions, ctx.rope, not ctx.inverse, None, None)[0], None, None, None, None
        gq, gk = _run(gq, gk, positions, ctx.rope, not ctx.inverse, None, None)
        return gq, gk, None, None, None

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        # linear: tangents are rotated as their tensors are (one that is absent stays so)
        positions, = ctx.saved_tensors
        tq, tk = (None if t is None else _run(t, None, positions, ctx.rope, ctx.inverse, None, None)[0] for t in (tq, tk))
        return (tq, tk) if ctx.two else tq


def _tracked(*ts):
    """Whether autograd has an interest in a call with these tensors, backward or forward."""
    for t in ts:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            return True
    # (there are no tangents outside of a dual level, where this costs a comparison)
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                                  for t in ts)


def fused_rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, rope: Rope, *,
               inverse: bool = False, out_q: torch.Tensor | None = None, out_k: torch.Tensor | None = None):
    """q and k (or None) with their heads turned by their tokens' positions: (q, k).

    q [T, Hq, D] or [B, L, Hq, D], k the same with its own heads; bf16, fp16 or fp32; any strides
    of tokens and heads (slices of a fused projection are read as they lie).  positions int32 or
    int64, one a token ([T] or [B, L]), or [.., axes] with a Rope of several axes; negative ones
    turn backwards.  fp32 between loads and stores, one rounding.  out_q / out_k may be q / k, and
    otherwise share no element with them or each other.
    inverse turns back, which is the gradient; autograd (once, backward or forward) goes through the
    call unless outputs are given.  D at most 256.
    """
    if not (q.is_cuda and positions.is_cuda and (k is None or k.is_cuda)):
        _lib.require_cuda(q, k, positions)
    if _tracked(q, k):
        if out_q is not None or out_k is not None:
            raise ValueError("fused_rope: out_q / out_k with inputs that require a gradient or carry a tangent")
        r = _Rotate.apply(q, k, positions, rope, bool(inverse))
        return r if k is not None else (r, None)
    return _run(q, k, positions, rope, bool(inverse), out_q, out_k)
