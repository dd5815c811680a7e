"""A key/value cache in pages, and attention over it, on the sm_100a library.

:class:`PagedKV` holds the keys and values of many streams in pages of one pool, for every layer:
chunks are appended (rotated on the way), branches share their parent's pages, streams give pages
back, the pool is compacted, and :meth:`PagedKV.attend` / ``paged_attention`` reads it.  The
streaming self-attention's own cache (integrate.py) is one contiguous buffer a stream with equal
heads; this is the form for many streams of uneven length, shared key heads and single tokens.

All state is device memory and every call is launches on the current stream, so a step over the
cache can be captured in a graph and replayed while the lengths grow.  Calls that change a cache
belong on one stream, or must be ordered by the caller.  Inference only.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .rope import Rope, _out, _positions, _rows

_DTYPES = {torch.bfloat16: _lib.FVB_BF16, torch.float16: _lib.FVB_F16}
_STATUS = {1: "no free pages left", 2: "a sequence outgrew its table row",
           4: "bad arguments (an index out of range or twice, a negative count, a branch that was not empty)"}


def _ints(t, n, what, name, device):
    if t.dtype != torch.int32 or t.dim() != 1 or (n is not None and t.numel() != n):
        raise ValueError(f"{name}: {what} must be int32 [{'n' if n is None else n}], got {t.dtype} {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name}: {what} is on {t.device}, the cache on {device}")
    return t if t.is_contiguous() else t.contiguous()


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
    are left as `out` had them (undefined in a new tensor).

    max_new, the most new tokens a sequence has, picks the kernel: with max_new * Hq / Hk <= 16
    the one for few rows.  It defaults to T (1 without cu_seqlens); any value gives the same
    results up to rounding.  What a page holds past a sequence's end is never seen, NaN or not.
    A NaN or an infinity among a sequence's own values can reach every row of the chunk that
    shares a tile with it, rows before it included.
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
    B = lens.numel()
    lens = _ints(lens, B, "lens", name, dev)
    if table.dim() != 2 or table.shape[0] != B or table.dtype != torch.int32 or table.device != dev:
        raise ValueError(f"{name}: table must be int32 [{B}, width] on {dev}, got {table.dtype} {tuple(table.shape)}")
    table = table if table.is_contiguous() else table.contiguous()
    if cu_seqlens is not None:
        cu_seqlens = _ints(cu_seqlens, B + 1, "cu_seqlens", name, dev)
    elif T != B:
        raise ValueError(f"{name}: {T} tokens of {B} sequences need cu_seqlens")
    if max_new is None:
        max_new = 1 if cu_seqlens is None else max(T, 1)
    elif max_new < 1:
        raise ValueError(f"{name}: max_new must be at least 1, got {max_new}")
    if Hk == 0 or Hq == 0 or Hq % Hk:
        raise ValueError(f"{name}: {Hq} query heads on {Hk} key heads")
    if q.stride(2) != 1 or (q.stride(0) | q.stride(1)) & 7 or q.data_ptr() & 15:
        q = q.clone(memory_format=torch.contiguous_format)
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
    if out is None:
        out = torch.empty((T, Hq, D), dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or out.stride(2) != 1 \
            or (out.stride(0) | out.stride(1)) & 7 or out.data_ptr() & 15:
        raise ValueError(f"{name}: out must be {q.dtype} [{T}, {Hq}, {D}] on {dev}, 16-byte aligned, strides "
                         f"multiples of 8")
    elif out.data_ptr() == q.data_ptr():
        raise ValueError(f"{name}: out cannot be q")
    nws = _workspace_bytes(max_new * (Hq // Hk) <= 16, D, dev.index)
    ws = torch.empty(nws, dtype=torch.uint8, device=dev)
    _lib.call_on(dev.index, "fvb_paged_attn", q.data_ptr(), q.stride(0), q.stride(1),
                 k_pages.data_ptr(), ks[0], ks[1], ks[2], v_pages.data_ptr(), vs[0], vs[1], vs[2],
                 table.data_ptr(), table.shape[1], lens.data_ptr(),
                 None if cu_seqlens is None else cu_seqlens.data_ptr(), T, B, Hq, Hk, D, P, page, max_new,
                 causal, 1.0 / math.sqrt(D) if sm_scale is None else sm_scale, dt, out.data_ptr(),
                 out.stride(0), out.stride(1), ws.data_ptr(), _lib.stream_of(q))
    return out


_WS: dict = {}


def _workspace_bytes(few, D, device):
    """fvb_paged_attn_workspace_bytes of few or many rows, asked for once a device."""
    n = _WS.get((few, D, device))
    if n is None:
        with torch.cuda.device(device):
            n = _lib.load().fvb_paged_attn_workspace_bytes(1 if few else 17, 1, 1, D)
        _WS[(few, D, device)] = n
    return n


class PagedKV:
    """Keys and values of `seqs` streams in pages.

    k, v    [layers, P, page, heads, D] bf16 or fp16; a page is contiguous, layers and pages may
            have any stride that is a multiple of 8
    table   int32 [seqs, width]: page numbers of each sequence, -1 for none
    lens    int32 [seqs]: tokens of each sequence
    refs    int32 [P]: how many sequences hold a page, 0 for free
    status  int32 [1]: what went wrong, see :meth:`check`

    The tensors are the state: read them, or hand in ones that hold one.  Free pages are given out
    lowest first in the order of sequences and of their pages.  A call on the device that cannot
    be done (no pages, an index out of range) changes nothing and is recorded in `status`.
    """

    def __init__(self, k, v, table, lens, refs):
        _lib.require_cuda(k, v, table, lens, refs)
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
        self.k, self.v, self.table, self.lens, self.refs = k, v, table, lens, refs
        self.page = page
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self.device = dev
        seqs, width = table.shape
        n = _lib.load().fvb_pages_workspace_bytes(seqs, P, seqs)
        self._ws = torch.empty(n, dtype=torch.uint8, device=dev)
        # what every step of the pages takes: the state, then its sizes
        self._state = (table.data_ptr(), lens.data_ptr(), refs.data_ptr(), self.status.data_ptr(), seqs, width, P,
                       page)
        self._pools = (k.data_ptr(), v.data_ptr(), k.shape[0], k.stride(0) * 2, k.stride(1) * 2, H * D * 2)

    @classmethod
    def empty(cls, layers: int, pages: int, page: int, heads: int, head_dim: int, seqs: int,
              width: int | None = None, dtype: torch.dtype = torch.bfloat16, device="cuda") -> "PagedKV":
        """A cache without tokens; width (pages a sequence can have) defaults to all of them."""
        shape = (layers, pages, page, heads, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device),
                   torch.full((seqs, pages if width is None else width), -1, dtype=torch.int32, device=device),
                   torch.zeros(seqs, dtype=torch.int32, device=device),
                   torch.zeros(pages, dtype=torch.int32, device=device))

    def check(self):
        """Waits for the device and raises what a step since the last check could not do."""
        s = int(self.status.item())
        if s:
            self.status.zero_()
            raise RuntimeError("PagedKV: " + "; ".join(m for bit, m in _STATUS.items() if s & bit))

    def _call(self, name, *args):
        _lib.call_on(self.device.index, name, *args, self._ws.data_ptr(), _lib.stream_of(self.table))

    def reserve(self, more: torch.Tensor):
        """Room for more[b] tokens (int32 [seqs]) behind every sequence; lens grow by them."""
        more = _ints(more, self.lens.numel(), "more", "PagedKV.reserve", self.device)
        self._call("fvb_pages_reserve", more.data_ptr(), *self._state)

    def fork(self, src: torch.Tensor, dst: torch.Tensor):
        """Sequence dst[i] becomes a branch of src[i] (int32 [n]; a parent may come several times,
        the branches are empty, distinct and no parents).  Full pages are shared; the tokens in a
        partly filled last page are copied, in every layer."""
        src = _ints(src, None, "src", "PagedKV.fork", self.device)
        dst = _ints(dst, src.numel(), "dst", "PagedKV.fork", self.device)
        if src.numel() > self.lens.numel():
            raise ValueError(f"PagedKV.fork: {src.numel()} branches of {self.lens.numel()} sequences")
        self._call("fvb_pages_fork", src.data_ptr(), dst.data_ptr(), src.numel(), *self._state, *self._pools)

    def release(self, seqs: torch.Tensor, pages: torch.Tensor | None = None):
        """Sequences (int32 [n], distinct) give back all their pages and become empty, or with
        `pages` (int32 [n]) that many of their first ones: a stream's oldest tokens.  Pages that
        other sequences hold stay."""
        seqs = _ints(seqs, None, "seqs", "PagedKV.release", self.device)
        if pages is not None:
            pages = _ints(pages, seqs.numel(), "pages", "PagedKV.release", self.device)
        self._call("fvb_pages_release", seqs.data_ptr(), None if pages is None else pages.data_ptr(), seqs.numel(),
                   *self._state)

    def compact(self):
        """Moves the pages in use to the front of the pool, so that its end is free."""
        self._call("fvb_pages_compact", *self._state, *self._pools)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, *,
               q: torch.Tensor | None = None, rope: Rope | None = None, positions: torch.Tensor | None = None,
               out_q: torch.Tensor | None = None):
        """Writes the last tokens of each sequence, those that reserve() made room for: k, v
        [T, heads, D] of all sequences, sequence b's at cu_seqlens[b] .. cu_seqlens[b + 1] (int32
        [seqs + 1]).  With a Rope, k is rotated on the way and so is q [T, Hq, D], which is
        returned; positions (as in fused_rope) default to the tokens' places in their sequences.
        Tokens past cu_seqlens[seqs] are ignored, and rows of out_q for them stay as they are."""
        name = "PagedKV.append"
        _lib.require_cuda(k, v, cu_seqlens, q, positions)
        H, D = self.k.shape[3:]
        k, v = _rows(k, "k", name), _rows(v, "v", name)
        T = k.shape[0]
        if k.shape != (T, H, D) or v.shape != (T, H, D):
            raise ValueError(f"{name}: k and v must be [T, {H}, {D}], got {tuple(k.shape)} and {tuple(v.shape)}")
        dt = self.k.dtype
        if k.dtype != dt or v.dtype != dt or k.device != self.device or v.device != self.device:
            raise ValueError(f"{name}: k and v must be {dt} on {self.device}")
        if not 0 <= layer < self.k.shape[0]:
            raise ValueError(f"{name}: layer {layer} of {self.k.shape[0]}")
        cu = _ints(cu_seqlens, self.lens.numel() + 1, "cu_seqlens", name, self.device)
        if q is None:
            if out_q is not None:
                raise ValueError(f"{name}: out_q without q")
            oq, qargs = None, (0, 0, 0, 0, 0, 0, 0)
        else:
            if rope is None:
                raise ValueError(f"{name}: q without a Rope has nothing to be done to it")
            if q.dtype != dt or q.device != self.device:
                raise ValueError(f"{name}: q must be {dt} on {self.device}")
            q3 = _rows(q, "q", name)
            if q3.shape[0] != T or q3.shape[2] != D:
                raise ValueError(f"{name}: q {tuple(q.shape)} does not match k {tuple(k.shape)}")
            oq, oq3 = _out(out_q, q, "out_q", name)
            s, so = q3.stride(), oq3.stride()
            qargs = (q3.data_ptr(), s[0], s[1], q3.shape[1], oq3.data_ptr(), so[0], so[1])
        if rope is None:
            if positions is not None:
                raise ValueError(f"{name}: positions without a Rope")
            rargs = (0, False, _DTYPES[dt], None, False, 1, None, None, 1.0)
        else:
            if rope.device != self.device or rope.rotary_dim > D:
                raise ValueError(f"{name}: {rope} on {rope.device} for heads of {D} on {self.device}")
            if positions is not None:
                positions = _positions(positions, rope, T, self.device, name)
            elif rope.axes > 1:
                raise ValueError(f"{name}: a Rope of {rope.axes} axes needs positions")
            rargs = (rope.rotary_dim, rope.half, _DTYPES[dt], None if positions is None else positions.data_ptr(),
                     positions is not None and positions.dtype == torch.int64, rope.axes, rope._freq, rope._axis,
                     rope.scale)
        ks, vs = k.stride(), v.stride()
        at = layer * self._pools[3]
        table, lens, _, _, seqs, width, pages, page = self._state
        _lib.call_on(self.device.index, "fvb_kv_append", *qargs, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0],
                     vs[1], H, T, D, *rargs, cu.data_ptr(), lens, table, seqs, width, pages, page,
                     self._pools[0] + at, self._pools[1] + at, self.k.stride(1), _lib.stream_of(k))
        return oq

    def attend(self, layer: int, q: torch.Tensor, cu_seqlens: torch.Tensor | None = None, *, causal: bool = True,
               sm_scale: float | None = None, max_new: int | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """paged_attention of q over one layer of this cache."""
        if not 0 <= layer < self.k.shape[0]:
            raise ValueError(f"PagedKV.attend: layer {layer} of {self.k.shape[0]}")
        return paged_attention(q, self.k[layer], self.v[layer], self.table, self.lens, cu_seqlens, causal=causal,
                               sm_scale=sm_scale, max_new=max_new, out=out)
