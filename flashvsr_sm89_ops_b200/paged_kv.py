"""A key/value cache in pages, and attention over it, on the sm_100a library.

:class:`PagedKV` holds the keys and values of many streams in pages of one pool, for every layer:
chunks are appended (rotated on the way), branches share their parent's pages, streams give pages
back, the pool is compacted, and :meth:`PagedKV.attend` / ``paged_attention`` reads it.  The
streaming self-attention's own cache (integrate.py) is one contiguous buffer a stream with equal
heads; this is the form for many streams of uneven length, shared key heads and single tokens.

All state is device memory and every call is launches on the current stream, so a step over the
cache can be captured in a graph and replayed while the lengths grow.  Calls that change a cache
belong on one stream, or must be ordered by the caller.  Inference only: inputs may require gradients,
but a backward pass through a result raises.
"""
from __future__ import annotations

import torch

from . import _lib
from .rope import _POS64, Rope, _apart, _out, _positions, _rows, _tracked

_DTYPES = {torch.bfloat16: _lib.FVB_BF16, torch.float16: _lib.FVB_F16}
_STATUS = {1: "no free pages left", 2: "a sequence outgrew its table row",
           4: "bad arguments (an index out of range or twice, a negative count or length, a branch that was not "
              "empty)",
           8: "tokens were not appended: the reserve() before them could not be done, or other sequences hold their "
              "page too"}


def _ints(t, n, what, name, index):
    s = t.shape
    if t.dtype != torch.int32 or len(s) != 1 or (n is not None and s[0] != n):
        raise ValueError(f"{name}: {what} must be int32 [{'n' if n is None else n}], got {t.dtype} {tuple(t.shape)}")
    if t.get_device() != index:
        raise ValueError(f"{name}: {what} is on {t.device}, the cache on cuda:{index}")
    return t if t.is_contiguous() else t.contiguous()


class _NoGradient(torch.autograd.Function):
    """A result of inputs that autograd follows.  It is what it is without them, but a backward pass through it
    raises where it would otherwise go by without these inputs' share."""

    @staticmethod
    def forward(ctx, name, y, *inputs):
        ctx.name = name
        ctx.mark_dirty(y)
        return y

    @staticmethod
    def backward(ctx, g):
        raise RuntimeError(f"{ctx.name} has no gradient (inference only)")


def _followed(name, y, *inputs):
    """y, the result of these inputs, for autograd: itself where that can be, else another name of it (a
    leaf, one of several views of a tensor)."""
    if not _tracked(*inputs):
        return y
    try:
        return _NoGradient.apply(name, y, *inputs)
    except RuntimeError:
        return _NoGradient.apply(name, y.detach(), *inputs)


def _beside(out, pools, shape, name):
    """Refuses an output that reaches into the pages of a layer."""
    Hk, D, P, page = shape
    at, end = out.data_ptr(), out.data_ptr() + 2 * (1 + sum((n - 1) * s for n, s in zip(out.shape, out.stride())))
    for p, sp, ss, sh in (pools[:4], pools[4:]):
        if out.numel() and P and at < p + 2 * ((P - 1) * sp + (page - 1) * ss + (Hk - 1) * sh + D) and p < end:
            raise ValueError(f"{name}: the output lies over the pages")


def _attend(name, q, dt, pools, shape, table, width, lens, B, cu_seqlens, causal, sm_scale, max_new, out, inputs):
    """The call itself.  pools: k, its three strides, v, its three strides; shape: Hk, D, P, page; inputs: what
    autograd could follow."""
    index = q.get_device()
    T, Hq, D = q.shape
    Hk, _, P, page = shape
    if cu_seqlens is not None:
        cu = _ints(cu_seqlens, B + 1, "cu_seqlens", name, index).data_ptr()
        max_new = max(T, 1) if max_new is None else max_new
    elif T != B:
        raise ValueError(f"{name}: {T} tokens of {B} sequences need cu_seqlens")
    else:
        cu = 0
        max_new = 1 if max_new is None else max_new
    if max_new < 1:
        raise ValueError(f"{name}: max_new must be at least 1, got {max_new}")
    if Hk == 0 or Hq == 0 or Hq % Hk:
        raise ValueError(f"{name}: {Hq} query heads on {Hk} key heads")
    st, sh, sd = q.stride()
    if sd != 1 or (st | sh) & 7 or st <= 0 or sh <= 0 or q.data_ptr() & 15:
        q = q.clone(memory_format=torch.contiguous_format)
        st, sh, _ = q.stride()
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        ot, oh = Hq * D, D
    else:
        if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
            raise ValueError(f"{name}: out must be {q.dtype} {tuple(q.shape)} on {q.device}")
        ot, oh, od = out.stride()
        if od != 1 or (ot | oh) & 7 or out.data_ptr() & 15:
            raise ValueError(f"{name}: out must be 16-byte aligned, with strides that are multiples of 8")
        _apart((out.data_ptr(), T, Hq, ot, oh, 2), [((q.data_ptr(), T, Hq, st, sh, 2), "q", False)], D, "out", name)
        _beside(out, pools, shape, name)
    few = max_new * (Hq // Hk) <= 16
    ws = torch.empty(_WS.get((few, D, index)) or _workspace_bytes(few, D, index), dtype=torch.uint8, device=q.device)
    _lib.call_on(index, "fvb_paged_attn",
                 _lib.PAGED_ATTN_ARGS(q.data_ptr(), st, sh, *pools, table, width, lens, cu, T, B, Hq, Hk, D, P, page,
                                      max_new, causal, D ** -0.5 if sm_scale is None else sm_scale, dt,
                                      out.data_ptr(), ot, oh, ws.data_ptr()), _lib.stream_of(q))
    return _followed(name, out, *inputs)


_WS: dict = {}


def _workspace_bytes(few, D, index):
    """fvb_paged_attn_workspace_bytes of few or many rows, asked for once a device."""
    with torch.cuda.device(index):
        n = _WS[(few, D, index)] = _lib.load().fvb_paged_attn_workspace_bytes(1 if few else 17, 1, 1, D)
    return n


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                    lens: torch.Tensor, cu_seqlens: torch.Tensor | None = None, *, causal: bool = True,
                    sm_scale: float | None = None, max_new: int | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of each sequence's new tokens over everything it has cached.

    q [T, Hq, D] bf16 or fp16: the new tokens of all sequences, sequence b's at
    cu_seqlens[b] .. cu_seqlens[b + 1] (int32 [B + 1]; None: one token each, T = B).  k_pages,
    v_pages [P, page, Hk, D], page a multiple of 16, any strides that are multiples of 8; query
    head h reads key head h // (Hq / Hk).  table int32 [B, width]; lens int32 [B] with the new
    tokens counted in.  Token i of n sees the first lens - n + i + 1 keys (causal) or all lens.
    D 64 or 128.  Returns [T, Hq, D]; a row that sees no key is 0, and rows past cu_seqlens[B]
    are left as `out` had them (undefined in a new tensor).  `out` shares no element with q or the
    pages.

    max_new, the most new tokens a sequence has, picks the kernel: with max_new * Hq / Hk <= 16
    the one for few rows.  It defaults to T (1 without cu_seqlens); any value gives the same
    results up to rounding.  What a page holds past a sequence's end is never seen, NaN or not.
    A NaN or an infinity among a sequence's own values can reach every row of the chunk that
    shares a tile with it, rows before it included.  A row that sees keys, but has only NaN or
    -inf for scores, is NaN.  Inference only: a backward pass through the result raises.
    """
    name = "paged_attention"
    _lib.require_cuda(q, k_pages, v_pages, table, lens, cu_seqlens)
    dt = _DTYPES.get(q.dtype)
    if dt is None:
        raise ValueError(f"{name}: expected bf16 or fp16, got {q.dtype}")
    if q.dim() != 3 or k_pages.dim() != 4 or v_pages.shape != k_pages.shape or q.shape[2] != k_pages.shape[3]:
        raise ValueError(f"{name}: q [T, Hq, D] and pages [P, page, Hk, D], got {tuple(q.shape)}, "
                         f"{tuple(k_pages.shape)}, {tuple(v_pages.shape)}")
    if k_pages.dtype != q.dtype or v_pages.dtype != q.dtype:
        raise ValueError(f"{name}: q is {q.dtype}, the pages {k_pages.dtype} and {v_pages.dtype}")
    T, Hq, D = q.shape
    P, page, Hk, _ = k_pages.shape
    dev = q.device
    if k_pages.device != dev or v_pages.device != dev:
        raise ValueError(f"{name}: q is on {dev}, the pages on {k_pages.device} and {v_pages.device}")
    index = dev.index
    B = lens.numel()
    lens = _ints(lens, B, "lens", name, index)
    if table.dim() != 2 or table.shape[0] != B or table.dtype != torch.int32 or table.device != dev:
        raise ValueError(f"{name}: table must be int32 [{B}, width] on {dev}, got {table.dtype} {tuple(table.shape)}")
    table = table if table.is_contiguous() else table.contiguous()
    # the stride of an axis of one is any number
    ks, vs = list(k_pages.stride()), list(v_pages.stride())
    for t, s in ((k_pages, ks), (v_pages, vs)):
        if s[3] != 1 or t.data_ptr() & 15:
            raise ValueError(f"{name}: pages must be 16-byte aligned with unit stride inside a head")
        for i, n in enumerate(t.shape[:3]):
            if n == 1:
                s[i] = D
            elif s[i] & 7 or s[i] <= 0:
                raise ValueError(f"{name}: strides of the pages must be positive multiples of 8, got {tuple(t.stride())}")
    return _attend(name, q, dt, (k_pages.data_ptr(), *ks[:3], v_pages.data_ptr(), *vs[:3]), (Hk, D, P, page),
                   table.data_ptr(), table.shape[1], lens.data_ptr(), B, cu_seqlens, causal, sm_scale, max_new, out,
                   (q, k_pages, v_pages))


class PagedKV:
    """Keys and values of `seqs` streams in pages.

    k, v    [layers, P, page, heads, D] bf16 or fp16; a page is contiguous, layers and pages may
            have any stride that is a multiple of 8
    table   int32 [seqs, width]: page numbers of each sequence, -1 for none
    lens    int32 [seqs]: tokens of each sequence
    refs    int32 [P]: how many sequences hold a page, 0 for free
    dropped int64 [seqs]: tokens that a sequence gave back at its start (all 0 if not handed in); its
            next token's position is dropped + its place.  0 again once it has no tokens
    status  int32 [1]: what went wrong, see :meth:`check`

    The tensors are the state: read them, or hand in ones that hold one.  Free pages are given out
    lowest first in the order of sequences and of their pages.  A call on the device that cannot
    be done (no pages, an index out of range) changes nothing and is recorded in `status`.  Behind a
    reserve() that could not be done, no append() writes anything until one is (`refused` int32 [1] is
    not 0): a step that found no room can be done again, and its results so far mean nothing.  At
    most 131072 sequences.
    """

    def __init__(self, k, v, table, lens, refs, dropped=None):
        _lib.require_cuda(k, v, table, lens, refs, dropped)
        if k.dim() != 5 or v.shape != k.shape or k.dtype not in _DTYPES or v.dtype != k.dtype:
            raise ValueError(f"PagedKV: k and v must be bf16 or fp16 [layers, P, page, heads, D], got "
                             f"{k.dtype} {tuple(k.shape)}, {v.dtype} {tuple(v.shape)}")
        _, P, page, H, D = k.shape
        if page < 1 or page % 16 or H < 1 or D % 8 or D < 8:
            raise ValueError(f"PagedKV: pages of a multiple of 16 tokens and heads of a multiple of 8 channels, got "
                             f"{tuple(k.shape)}")
        for t in (k, v):
            if t.stride()[2:] != (H * D, D, 1) and t.numel() or t.stride(0) % 8 or t.stride(1) % 8 \
                    or t.data_ptr() & 15:
                raise ValueError("PagedKV: a page must be contiguous and 16-byte aligned")
        if k.stride() != v.stride():
            raise ValueError("PagedKV: k and v must have the same strides")
        dev = k.device
        if table.dim() != 2 or table.dtype != torch.int32 or not table.is_contiguous() or table.device != dev:
            raise ValueError(f"PagedKV: table must be contiguous int32 [seqs, width] on {dev}")
        for t, n, what in ((lens, table.shape[0], "lens"), (refs, P, "refs")):
            if t.dtype != torch.int32 or t.shape != (n,) or not t.is_contiguous() or t.device != dev:
                raise ValueError(f"PagedKV: {what} must be contiguous int32 [{n}] on {dev}")
        if v.device != dev:
            raise ValueError(f"PagedKV: k is on {dev}, v on {v.device}")
        if dropped is None:
            dropped = torch.zeros(table.shape[0], dtype=torch.int64, device=dev)
        elif dropped.dtype != torch.int64 or dropped.shape != lens.shape or not dropped.is_contiguous() \
                or dropped.device != dev:
            raise ValueError(f"PagedKV: dropped must be contiguous int64 [{table.shape[0]}] on {dev}")
        self._tensors = (k, v, table, lens, refs, *torch.zeros(2, dtype=torch.int32, device=dev).split(1), dropped)
        self._bind()

    def _bind(self):
        k, v, table, lens, refs, status, refused, dropped = self._tensors
        _, P, page, H, D = k.shape
        self.page = page
        self.device = dev = k.device
        seqs, width = table.shape
        n = _lib.load().fvb_pages_workspace_bytes(seqs, P)
        self._ws = torch.empty(n, dtype=torch.uint8, device=dev)
        self._pools = (k.data_ptr(), v.data_ptr(), k.shape[0], k.stride(0) * 2, k.stride(1) * 2, H * D * 2)
        # what every step of the pages takes
        self._pages = _lib.PAGES(table.data_ptr(), lens.data_ptr(), refs.data_ptr(), status.data_ptr(), seqs, width, P,
                                 page, *self._pools, self._ws.data_ptr(), refused=refused.data_ptr(),
                                 dropped=dropped.data_ptr())
        # and every append and attention
        self._index, self._dt, self._dtype = k.get_device(), _DTYPES[k.dtype], k.dtype
        self._shape = (H, D, P, page)
        self._strides = (k.stride(1) if P > 1 else page * H * D, H * D, D)
        self._tail = (lens.data_ptr(), table.data_ptr(), seqs, width, P, page)
        self._room = (refused.data_ptr(), refs.data_ptr(), status.data_ptr(), dropped.data_ptr())

    # a copy has tensors, and so addresses and a workspace, of its own
    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k != "_ws"}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._bind()

    @classmethod
    def empty(cls, layers: int, pages: int, page: int, heads: int, head_dim: int, seqs: int,
              width: int | None = None, dtype: torch.dtype = torch.bfloat16, device="cuda") -> "PagedKV":
        """A cache without tokens; width (pages a sequence can have) defaults to all of them."""
        shape = (layers, pages, page, heads, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device),
                   torch.full((seqs, pages if width is None else width), -1, dtype=torch.int32, device=device),
                   torch.zeros(seqs, dtype=torch.int32, device=device),
                   torch.zeros(pages, dtype=torch.int32, device=device))

    # the calls hold the addresses of these, so they can be written to but not replaced
    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    table = property(lambda self: self._tensors[2])
    lens = property(lambda self: self._tensors[3])
    refs = property(lambda self: self._tensors[4])
    status = property(lambda self: self._tensors[5])
    refused = property(lambda self: self._tensors[6])
    dropped = property(lambda self: self._tensors[7])

    def check(self):
        """Waits for the device and raises what a step since the last check could not do."""
        s = int(self.status.item())
        if s:
            self.status.zero_()
            raise RuntimeError("PagedKV: " + "; ".join(m for bit, m in _STATUS.items() if s & bit))

    def reserve(self, more: torch.Tensor):
        """Room for more[b] tokens (int32 [seqs]) behind every sequence; lens grow by them."""
        more = _ints(more, self._tail[2], "more", "PagedKV.reserve", self._index)
        _lib.call_on(self._index, "fvb_pages_reserve", self._pages, more.data_ptr(), _lib.stream_of(more))

    def fork(self, src: torch.Tensor, dst: torch.Tensor):
        """Sequence dst[i] becomes a branch of src[i] (int32 [n]; a parent may come several times,
        the branches are empty, distinct and no parents).  Full pages are shared; the tokens in a
        partly filled last page are copied, in every layer: what reserve() made room for is appended
        first."""
        src = _ints(src, None, "src", "PagedKV.fork", self._index)
        n = src.shape[0]
        dst = _ints(dst, n, "dst", "PagedKV.fork", self._index)
        _lib.call_on(self._index, "fvb_pages_fork", self._pages, src.data_ptr(), dst.data_ptr(), n,
                     _lib.stream_of(src))

    def release(self, seqs: torch.Tensor, pages: torch.Tensor | None = None):
        """Sequences (int32 [n], distinct) give back all their pages and become empty, or with
        `pages` (int32 [n]) that many of their first ones: a stream's oldest tokens.  Pages that
        other sequences hold stay.  What a sequence keeps is as it was rotated, and its next tokens'
        positions go on from there (`dropped`)."""
        seqs = _ints(seqs, None, "seqs", "PagedKV.release", self._index)
        n = seqs.shape[0]
        if pages is not None:
            pages = _ints(pages, n, "pages", "PagedKV.release", self._index)
        _lib.call_on(self._index, "fvb_pages_release", self._pages, seqs.data_ptr(),
                     None if pages is None else pages.data_ptr(), n, _lib.stream_of(seqs))

    def compact(self):
        """Moves the pages in use to the front of the pool, so that its end is free."""
        _lib.call_on(self._index, "fvb_pages_compact", self._pages, _lib.stream_of(self.table))

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, *,
               q: torch.Tensor | None = None, rope: Rope | None = None, positions: torch.Tensor | None = None,
               out_q: torch.Tensor | None = None):
        """Writes the last tokens of each sequence, those that reserve() made room for: k, v
        [T, heads, D] of all sequences, sequence b's at cu_seqlens[b] .. cu_seqlens[b + 1] (int32
        [seqs + 1]).  With a Rope, k is rotated on the way and so is q [T, Hq, D], which is
        returned; positions (as in fused_rope) default to the tokens' places in their sequences, tokens
        that release() dropped at their start counted.
        Tokens past cu_seqlens[seqs] are ignored, and rows of out_q for them stay as they are.  If
        the last reserve() could not be done, nothing is written, out_q neither, and check() raises; so
        it does where a token's page belongs to other sequences too, which is left as it is."""
        name = "PagedKV.append"
        index, dt = self._index, self._dtype
        H, D, P, page = self._shape
        if not (k.is_cuda and v.is_cuda and cu_seqlens.is_cuda):
            _lib.require_cuda(k, v, cu_seqlens)
        k, T, Hk, Dk, kt, kh = _rows(k, "k", name)
        v, Tv, Hv, Dv, vt, vh = _rows(v, "v", name)
        if Hk != H or Dk != D or Tv != T or Hv != H or Dv != D:
            raise ValueError(f"{name}: k and v must be [T, {H}, {D}], got {tuple(k.shape)} and {tuple(v.shape)}")
        if k.dtype != dt or v.dtype != dt or k.get_device() != index or v.get_device() != index:
            raise ValueError(f"{name}: k and v must be {dt} on {self.device}")
        if not 0 <= layer < self._pools[2]:
            raise ValueError(f"{name}: layer {layer} of {self._pools[2]}")
        lens, table, seqs, width, P, page = self._tail
        cu = _ints(cu_seqlens, seqs + 1, "cu_seqlens", name, index)
        if q is None:
            if out_q is not None:
                raise ValueError(f"{name}: out_q without q")
            oq, qargs = None, (0, 0, 0, 0, 0, 0, 0)
        else:
            if rope is None:
                raise ValueError(f"{name}: q without a Rope has nothing to be done to it")
            if q.dtype != dt or q.get_device() != index:
                raise ValueError(f"{name}: q must be {dt} on {self.device}")
            q3, Tq, Hq, Dq, st, sh = _rows(q, "q", name)
            if Tq != T or Dq != D:
                raise ValueError(f"{name}: q {tuple(q.shape)} does not match k {tuple(k.shape)}")
            oq, ot, oh = _out(out_q, q, "out_q", name)
            qargs = (q3.data_ptr(), st, sh, Hq, oq.data_ptr(), ot, oh)
            if out_q is not None:
                _apart((oq.data_ptr(), T, Hq, ot, oh, 2), [((q3.data_ptr(), T, Hq, st, sh, 2), "q", True),
                                                           ((k.data_ptr(), T, H, kt, kh, 2), "k", False),
                                                           ((v.data_ptr(), T, H, vt, vh, 2), "v", False)], D, "out_q", name)
                kp, vp, _, layer_bytes, _, _ = self._pools
                at = layer * layer_bytes
                _beside(oq, (kp + at, *self._strides, vp + at, *self._strides), self._shape, name)
        if rope is None:
            if positions is not None:
                raise ValueError(f"{name}: positions without a Rope")
            rargs = (0, 0, self._dt, 0, 0, 1, 0, 0, 1.0)
        else:
            if rope.index != index or rope.rotary_dim > D:
                raise ValueError(f"{name}: {rope} on {rope.device} for heads of {D} on {self.device}")
            if positions is None:
                if rope.axes > 1:
                    raise ValueError(f"{name}: a Rope of {rope.axes} axes needs positions")
                pos, pos64 = 0, 0
            else:
                positions = _positions(positions, rope, T, index, name)
                pos, pos64 = positions.data_ptr(), _POS64[positions.dtype]
            rargs = (rope.rotary_dim, rope.half, self._dt, pos, pos64, rope.axes, rope._freq, rope._axis, rope.scale)
        kp, vp, _, layer_bytes, _, _ = self._pools
        at = layer * layer_bytes
        _lib.call_on(index, "fvb_kv_append",
                     _lib.KV_APPEND_ALL(*qargs, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, H, T, D, *rargs,
                                        cu.data_ptr(), lens, table, seqs, width, P, page, kp + at, vp + at,
                                        self._strides[0], *self._room), _lib.stream_of(k))
        return None if oq is None else _followed(name, oq, q, k, v)

    def attend(self, layer: int, q: torch.Tensor, cu_seqlens: torch.Tensor | None = None, *, causal: bool = True,
               sm_scale: float | None = None, max_new: int | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """paged_attention of q over one layer of this cache.  With cu_seqlens, max_new says where there are few
        new tokens a sequence (1: single ones): without it the kernel for many rows is taken."""
        name = "PagedKV.attend"
        if not 0 <= layer < self._pools[2]:
            raise ValueError(f"{name}: layer {layer} of {self._pools[2]}")
        if not q.is_cuda:
            _lib.require_cuda(q)
        if q.dtype != self._dtype or q.get_device() != self._index or q.dim() != 3 or q.shape[2] != self._shape[1]:
            raise ValueError(f"{name}: q must be {self._dtype} [T, Hq, {self._shape[1]}] on {self.device}, got {q.dtype} "
                             f"{tuple(q.shape)} on {q.device}")
        kp, vp, _, layer_bytes, _, _ = self._pools
        at, s = layer * layer_bytes, self._strides
        lens, table, seqs, width, _, _ = self._tail
        return _attend(name, q, self._dt, (kp + at, *s, vp + at, *s), self._shape, table, width, lens, seqs,
                       cu_seqlens, causal, sm_scale, max_new, out, (q,))
