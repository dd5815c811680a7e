"""Rotary positions, the paged cache and attention over it, against their definitions in 64 bits.

Tolerances are bounds of the roundings that the kernels make, written out at `_attend_bound` and
`_rope_bound`; page tables, lengths and copies have to be equal.
"""
import math
import random

import pytest
import torch

import flashvsr_sm89_ops_b200 as ops
from flashvsr_sm89_ops_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step
# half of the smallest step: below its normal range (2^-14 in fp16) a type's step no longer shrinks
# with the value, so a rounding there is off by up to this and not by U of the value
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


@pytest.fixture(autouse=True)
def no_timeouts():
    yield
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _cu(new):
    return _i32([sum(new[:i]) for i in range(len(new) + 1)])


# ------------------------------------------------------------------------------- rope
def _rope_64(x, positions, rot, half, freqs, axis, scale, inverse):
    """x [T, H, D]; positions [T, axes]; freqs in 64 bits."""
    x = x.double()
    ang = positions.double()[:, axis] * freqs
    c, s = torch.cos(ang)[:, None] * scale, torch.sin(ang)[:, None] * scale
    if inverse:
        s = -s
    y = x.clone()
    a = x[..., :rot // 2] if half else x[..., 0:rot:2]
    b = x[..., rot // 2:rot] if half else x[..., 1:rot:2]
    ya, yb = a * c - b * s, b * c + a * s
    if half:
        y[..., :rot // 2], y[..., rot // 2:rot] = ya, yb
    else:
        y[..., 0:rot:2], y[..., 1:rot:2] = ya, yb
    m = x.abs() * 0
    both = (a.abs() + b.abs()) * scale
    if half:
        m[..., :rot // 2], m[..., rot // 2:rot] = both, both
    else:
        m[..., 0:rot:2], m[..., 1:rot:2] = both, both
    return y, m


def _rope_bound(y, both, dtype):
    """Half a step of the result, and of a c - b s in fp32: the angle's rounding (pi 2^-24), that
    of sine and cosine (2^-22), their factor and the two products (3 x 2^-24): below 1e-6."""
    return U[dtype] * y.abs() * (1 + 1e-5) + 1e-6 * both + TINY[dtype]


def _freqs(dims, theta=10000.0):
    f = torch.cat([theta ** (-torch.arange(0, d, 2, dtype=torch.float64) / d) for d in dims if d])
    return f.to(DEV), torch.tensor([a for a, d in enumerate(dims) for _ in range(d // 2)], device=DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("T,Hq,Hk,D,rot", [(1, 12, 12, 128, 128), (7, 5, 1, 64, 32), (300, 8, 2, 96, 70),
                                           (2500, 3, 3, 80, 40), (33, 1, 1, 6, 2), (5, 2, 1, 256, 256),
                                           (3, 4, 2, 64, 0), (20000, 2, 1, 16, 16)])
@pytest.mark.parametrize("inverse", [False, True])
def test_rope(T, Hq, Hk, D, rot, half, dtype, inverse):
    g = _gen(T + D + rot)
    # slices of a fused projection; with an odd pitch the vectors cannot be used
    pitch = (Hq + Hk) * D + (1 if T == 300 else 0)
    x = torch.randn(T, pitch, device=DEV, generator=g).to(dtype)
    q = x[:, :Hq * D].unflatten(1, (Hq, D))
    k = x[:, Hq * D:(Hq + Hk) * D].unflatten(1, (Hk, D))
    pos = torch.randint(-50, 200000, (T,), device=DEV, generator=g)
    if T % 2:
        pos = pos.int()
    rope = ops.Rope(rot, layout="half" if half else "interleaved")
    oq, ok = ops.fused_rope(q, k, pos, rope, inverse=inverse)
    f, axis = _freqs((rot,)) if rot else (torch.zeros(0, device=DEV), torch.zeros(0, device=DEV, dtype=torch.long))
    for a, y in ((q, oq), (k, ok)):
        want, both = _rope_64(a, pos[:, None], rot, half, f, axis, 1.0, inverse)
        assert y.shape == a.shape and y.dtype == dtype and y.is_contiguous()
        assert ((y.double() - want).abs() <= _rope_bound(want, both, dtype)).all()
        assert torch.equal(y[..., rot:], a[..., rot:])


def test_rope_far_positions():
    """Angles keep fp32 precision at positions where the product in fp32 has none left."""
    pos = torch.tensor([0, 1, -1, 2 ** 20 + 1, 2 ** 31 - 1, -2 ** 31, 2 ** 40 + 12345], device=DEV)
    x = torch.randn(7, 1, 64, device=DEV, generator=_gen(1))
    y, _ = ops.fused_rope(x, None, pos, ops.Rope(64))
    # exact: whole turns dropped in integers of 200 bits
    pi2 = 2 * 3141592653589793238462643383279502884197169399375105820974944592307816406286
    for t, p in enumerate(pos.tolist()):
        for i in range(32):
            w = 10000.0 ** (-2 * i / 64)
            num, den = w.as_integer_ratio()
            ang = (p * num * 10 ** 75) % (pi2 * den) / (den * 10 ** 75)
            a, b = x[t, 0, 2 * i].item(), x[t, 0, 2 * i + 1].item()
            # the frequency is held to 2^-53 of itself: beyond 2^31 that is what is left
            tol = (1e-6 + abs(p) * w * 2.0 ** -52) * (abs(a) + abs(b))
            assert abs(y[t, 0, 2 * i].item() - (a * math.cos(ang) - b * math.sin(ang))) <= tol
            assert abs(y[t, 0, 2 * i + 1].item() - (b * math.cos(ang) + a * math.sin(ang))) <= tol


def test_rope_three_axes_is_the_dit_rotation():
    """Frame, row and column positions: the table that the DiT's own rope_apply takes."""
    from flashvsr_sm89_ops_b200 import wan_video_dit as W
    f, h, w, heads = 2, 16, 24, 12
    freqs = W.grid_freqs(W.precompute_freqs_cis_3d(128), f, h, w, f0=6).to(DEV)
    x = torch.randn(1, f * h * w, heads * 128, device=DEV, generator=_gen(3))
    want = W.rope_apply(x.double(), freqs, heads)
    grid = torch.stack(torch.meshgrid(torch.arange(6, 6 + f), torch.arange(h), torch.arange(w), indexing="ij"), -1)
    rope = ops.Rope(128, axes=(44, 42, 42))
    y, _ = ops.fused_rope(x.unflatten(2, (heads, 128)), None, grid.view(1, -1, 3).to(DEV), rope)
    assert (y.flatten(2).double() - want).abs().max() <= 1e-6 * 2 * x.abs().max() + 2.0 ** -24 * want.abs().max()


@pytest.mark.parametrize("scaling,kw", [("linear", {}), ("ntk", {}), ("yarn", {"original_len": 4096})])
def test_rope_scalings(scaling, kw):
    d, theta, s = 128, 10000.0, 4.0
    i = torch.arange(d // 2, dtype=torch.float64)
    f = theta ** (-2 * i / d)
    m = 1.0
    if scaling == "linear":
        f = f / s
    elif scaling == "ntk":
        f = (theta * s ** (d / (d - 2))) ** (-2 * i / d)
    else:
        turns = 4096 * f / (2 * math.pi)
        # the ramp lies between the pairs that turn 32 times and once; both ends are rounded outwards
        lo = torch.nonzero(turns > 32).max().item()
        hi = torch.nonzero(turns < 1).min().item()
        r = ((i - lo) / (hi - lo)).clamp(0, 1)
        f = f * (1 - r) + f / s * r
        m = 0.1 * math.log(s) + 1
    x = torch.randn(50, 2, d, device=DEV, generator=_gen(5))
    pos = torch.arange(0, 16000, 320, device=DEV)
    y, _ = ops.fused_rope(x, None, pos, ops.Rope(d, scaling=scaling, factor=s, **kw))
    want, both = _rope_64(x, pos[:, None], d, False, f.to(DEV), torch.zeros(d // 2, dtype=torch.long, device=DEV), m, False)
    assert ((y.double() - want).abs() <= _rope_bound(want, both, torch.float32)).all()


def test_rope_gradients():
    g = _gen(7)
    q = torch.randn(9, 4, 32, device=DEV, generator=g).requires_grad_()
    k = torch.randn(9, 2, 32, device=DEV, generator=g).requires_grad_()
    pos = torch.randint(0, 5000, (9,), device=DEV, generator=g)
    rope = ops.Rope(24, layout="half", scaling="yarn", factor=2.0, original_len=512)
    oq, ok = ops.fused_rope(q, k, pos, rope)
    wq, wk = torch.randn_like(oq), torch.randn_like(ok)
    ((oq * wq).sum() + (ok * wk).sum()).backward()
    # the rotation is linear: its gradient is its transpose, and differences are exact up to rounding
    for x, w in ((q, wq), (k, wk)):
        iq, _ = ops.fused_rope(w, None, pos, rope, inverse=True)
        assert torch.equal(x.grad, iq)
        d = torch.randn_like(x)
        with torch.no_grad():
            yd = ops.fused_rope(d, None, pos, rope)[0].double()
        lhs, rhs = (yd * w.double()).sum(), (d.double() * x.grad.double()).sum()
        # both sums have numel terms, each off by at most 2e-6 of its factors
        assert (lhs - rhs).abs() <= 2 * 2e-6 * rope.scale * 2 * (d.abs().max() * w.abs().max()).double() * d.numel()
    # one tensor alone, and no gradient for what needs none
    q.grad = None
    ops.fused_rope(q, None, pos, rope)[0].backward(wq)
    assert torch.equal(q.grad, ops.fused_rope(wq, None, pos, rope, inverse=True)[0])
    a, b = ops.fused_rope(q, k.detach(), pos, rope)
    a.sum().backward()


def test_rope_in_place_and_out():
    x = torch.randn(2, 40, 6, 64, device=DEV, generator=_gen(9)).bfloat16()
    pos = torch.arange(80, device=DEV, dtype=torch.int32).view(2, 40)
    for layout in ("half", "interleaved"):
        rope = ops.Rope(32, layout=layout)
        want, _ = ops.fused_rope(x, None, pos, rope)
        y = x.clone()
        r, none = ops.fused_rope(y, None, pos, rope, out_q=y)
        assert r is y and none is None and torch.equal(y, want)
        wide = torch.full((2, 40, 6, 80), 7.0, device=DEV, dtype=torch.bfloat16)
        ops.fused_rope(x, None, pos, rope, out_q=wide[..., :64])
        assert torch.equal(wide[..., :64], want) and (wide[..., 64:] == 7).all()
    z = torch.zeros(0, 3, 64, device=DEV)
    assert ops.fused_rope(z, z, pos.view(-1)[:0], rope)[0].shape == (0, 3, 64)


# ------------------------------------------------------------------------------- pages, in plain Python
class Book:
    """The page tables, a page at a time."""

    def __init__(self, table, lens, refs, page):
        self.table, self.lens, self.refs, self.page = table, lens, refs, page

    @classmethod
    def of(cls, kv):
        return cls(kv.table.tolist(), kv.lens.tolist(), kv.refs.tolist(), kv.page)

    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def pages(self, n):
        return -(-n // self.page)

    def reserve(self, more):
        for b, n in enumerate(more):
            for j in range(self.pages(self.lens[b]), self.pages(self.lens[b] + n)):
                self.table[b][j] = self.take()
            self.lens[b] += n

    def fork(self, src, dst):
        copies = []
        for a, d in zip(src, dst):
            for j in range(self.lens[a] // self.page):
                self.table[d][j] = self.table[a][j]
                self.refs[self.table[a][j]] += 1
            self.lens[d] = self.lens[a]
        for a, d in zip(src, dst):
            if self.lens[a] % self.page:
                j = self.lens[a] // self.page
                self.table[d][j] = self.take()
                copies.append((self.table[a][j], self.table[d][j], self.lens[a] % self.page))
        return copies

    def release(self, seqs, pages=None):
        for i, b in enumerate(seqs):
            have = self.pages(self.lens[b])
            gone = have if pages is None else min(pages[i], have)
            for p in self.table[b][:gone]:
                self.refs[p] -= 1
            w = len(self.table[b])
            self.table[b] = (self.table[b][gone:have] + [-1] * w)[:w]
            self.lens[b] = max(self.lens[b] - gone * self.page, 0)

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        holes = [p for p in range(used) if not self.refs[p]]
        movers = [p for p in range(used, len(self.refs)) if self.refs[p]]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return to

    def check(self, kv):
        assert kv.table.tolist() == self.table
        assert kv.lens.tolist() == self.lens
        assert kv.refs.tolist() == self.refs


def _fill(kv, seed):
    g = _gen(seed)
    for t in (kv.k, kv.v):
        for layer in t:
            layer.normal_(generator=g)


def _tokens(kv, b):
    """What sequence b holds, [layers, len, heads, D] of k and v."""
    n = kv.lens[b].item()
    at = torch.arange(n, device=DEV)
    rows = kv.table[b].long()[at // kv.page]
    return kv.k[:, rows, at % kv.page].clone(), kv.v[:, rows, at % kv.page].clone()


@pytest.mark.parametrize("page,seqs,pages,width", [(16, 5, 60, 20), (48, 3, 2100, 1300), (128, 40, 9000, 30),
                                                   (16, 1300, 5000, 4)])
def test_pages_follow_the_book(page, seqs, pages, width):
    """Random steps; tables, lengths and reference counts equal, and every sequence keeps its tokens."""
    r = random.Random(page * seqs)
    kv = ops.PagedKV.empty(2, pages, page, 1, 8, seqs, width, dtype=torch.float16)
    _fill(kv, 1)
    book = Book.of(kv)
    if page == 48:  # past 1024 pages in one call, and past one pass over the list of free pages
        more = [page * 1250 + 7, 0, 5]
        kv.reserve(_i32(more))
        book.reserve(more)
        book.check(kv)
    for step in range(12):
        more = [r.choice((0, 1, page // 2, page, 3 * page - 1)) for _ in range(seqs)]
        more = [n if book.lens[b] + n <= width * page and r.random() < 0.7 else 0 for b, n in enumerate(more)]
        if sum(book.pages(book.lens[b] + n) - book.pages(book.lens[b]) for b, n in enumerate(more)) \
                <= sum(x == 0 for x in book.refs):
            kv.reserve(_i32(more))
            book.reserve(more)
            book.check(kv)
        held = [b for b in range(seqs) if book.lens[b]]
        drop = r.sample(held, min(len(held), 1 + seqs // 8))
        if drop and step % 2:
            count = [r.choice((0, 1, 2, 1000)) for _ in drop] if r.random() < 0.5 else None
            kv.release(_i32(drop), None if count is None else _i32(count))
            book.release(drop, count)
            book.check(kv)
        empty = [b for b in range(seqs) if not book.lens[b]]
        held = [b for b in range(seqs) if book.lens[b]]
        if empty and held:
            dst = r.sample(empty, min(len(empty), 1 + seqs // 6))
            src = [r.choice(held) for _ in dst]
            if sum(book.lens[a] % page > 0 for a in src) <= sum(x == 0 for x in book.refs):
                before = [_tokens(kv, a) for a in src]
                kv.fork(_i32(src), _i32(dst))
                book.fork(src, dst)
                book.check(kv)
                for d, (k, v) in zip(dst, before):
                    k2, v2 = _tokens(kv, d)
                    assert torch.equal(k, k2) and torch.equal(v, v2)
        if step % 3 == 2:
            some = r.sample(range(seqs), min(seqs, 20))
            before = [_tokens(kv, b) for b in some]
            kv.compact()
            book.compact()
            book.check(kv)
            for b, (k, v) in zip(some, before):
                k2, v2 = _tokens(kv, b)
                assert torch.equal(k, k2) and torch.equal(v, v2)
    kv.check()


@pytest.mark.parametrize("dtype,H,D,page", [(torch.bfloat16, 12, 128, 128), (torch.float16, 3, 64, 16)])
def test_pages_copies_and_nothing_else(dtype, H, D, page):
    """Every byte of both pools after a fork and a compaction, in a strided pool of several layers."""
    both = torch.empty(3, 40, 2, page, H, D, device=DEV, dtype=dtype)  # k and v of a page side by side
    both.normal_(generator=_gen(2))
    kv = ops.PagedKV(both[:, :, 0], both[:, :, 1], torch.full((6, 8), -1, dtype=torch.int32, device=DEV),
                     _i32([0] * 6), _i32([1, 0] * 20))
    book = Book.of(kv)
    more = [2 * page + 5, page, 0, 0, 0, 0]
    kv.reserve(_i32(more))
    book.reserve(more)
    want_k, want_v = kv.k.clone(), kv.v.clone()
    kv.fork(_i32([0, 1, 0]), _i32([4, 2, 3]))
    for a, b, n in book.fork([0, 1, 0], [4, 2, 3]):
        want_k[:, b, :n], want_v[:, b, :n] = want_k[:, a, :n], want_v[:, a, :n]
    book.check(kv)
    assert torch.equal(kv.k, want_k) and torch.equal(kv.v, want_v)
    kv.compact()
    for a, b in book.compact().items():
        want_k[:, b], want_v[:, b] = want_k[:, a], want_v[:, a]
    book.check(kv)
    assert torch.equal(kv.k, want_k) and torch.equal(kv.v, want_v)
    kv.check()


def test_pages_refuse_what_cannot_be_done():
    """Nothing changes, the reason is raised by check(), and the cache goes on."""
    kv = ops.PagedKV.empty(1, 8, 16, 1, 8, 4, 5)
    kv.reserve(_i32([20, 16, 0, 0]))
    book = Book([[0, 1, -1, -1, -1], [2, -1, -1, -1, -1], [-1] * 5, [-1] * 5], [20, 16, 0, 0], [1, 1, 1, 0, 0, 0, 0, 0], 16)
    book.check(kv)
    cases = [(lambda: kv.reserve(_i32([0, 0, 80, 16])), "no free pages"),
             (lambda: kv.reserve(_i32([61, 0, 0, 0])), "table row"),
             (lambda: kv.reserve(_i32([0, -1, 0, 0])), "bad arguments"),
             (lambda: kv.reserve(_i32([2 ** 31 - 1, 0, 0, 0])), "bad arguments"),
             (lambda: kv.fork(_i32([0]), _i32([1])), "bad arguments"),        # not empty
             (lambda: kv.fork(_i32([0, 0]), _i32([2, 2])), "bad arguments"),  # twice
             (lambda: kv.fork(_i32([0]), _i32([4])), "bad arguments"),
             (lambda: kv.fork(_i32([-1]), _i32([2])), "bad arguments"),
             (lambda: kv.fork(_i32([2]), _i32([2])), "bad arguments"),        # its own parent
             (lambda: kv.release(_i32([0, 0])), "bad arguments"),
             (lambda: kv.release(_i32([9])), "bad arguments"),
             (lambda: kv.release(_i32([0]), _i32([-1])), "bad arguments")]
    for call, why in cases:
        call()
        with pytest.raises(RuntimeError, match=why):
            kv.check()
        book.check(kv)
        kv.check()
    kv.lens[2] = -5  # a state that was handed in broken
    for call in (lambda: kv.reserve(_i32([0] * 4)), lambda: kv.fork(_i32([2]), _i32([3]))):
        call()
        with pytest.raises(RuntimeError, match="bad arguments"):
            kv.check()
    kv.release(_i32([2]))
    book.check(kv)
    kv.reserve(_i32([0, 0, 80, 0]))
    book.reserve([0, 0, 80, 0])
    kv.fork(_i32([0]), _i32([3]))  # its last page is partly filled, and none is free
    with pytest.raises(RuntimeError, match="no free pages"):
        kv.check()
    book.check(kv)
    kv.fork(_i32([1]), _i32([3]))  # a full one needs none
    book.fork([1], [3])
    kv.release(_i32([]))
    book.check(kv)
    kv.check()


# ------------------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hk,D,rot,layout,page", [(12, 12, 128, 128, "interleaved", 128), (6, 2, 64, 64, "half", 16),
                                                     (4, 1, 72, 20, "interleaved", 48), (0, 3, 64, 0, None, 32),
                                                     (2, 2, 96, 50, "half", 16)])
def test_append(Hq, Hk, D, rot, layout, page, dtype):
    new, had = [3, 0, 130, 1, 40], [15, 20, 0, 64, 1000]
    B, T = len(new), sum(new)
    kv = ops.PagedKV.empty(2, 120, page, Hk, D, B, 70, dtype=dtype)
    _fill(kv, 3)
    kv.reserve(_i32(had))
    kv.reserve(_i32(new))
    g = _gen(4)
    pad = 4  # tokens behind the last sequence
    x = torch.randn(T + pad, (Hq + 2 * Hk) * D, device=DEV, generator=g).to(dtype)
    q, k, v = (t.unflatten(1, (-1, D)) if t.shape[1] else None
               for t in x.split((Hq * D, Hk * D, Hk * D), 1))
    want_k, want_v = kv.k.clone(), kv.v.clone()
    rope = ops.Rope(rot, layout=layout) if layout else None
    out = torch.full((T + pad, Hq, D), 3.0, device=DEV, dtype=dtype) if Hq else None
    got = kv.append(1, k, v, _cu(new), q=q, rope=rope, out_q=out)
    pos = torch.cat([torch.arange(h, h + n) for h, n in zip(had, new)]).to(DEV)
    seq = torch.cat([torch.full((n,), b) for b, n in enumerate(new)]).to(DEV)
    rows = kv.table.long()[seq, pos // page]
    want_v[1, rows, pos % page] = v[:T]
    if rope is None:
        want_k[1, rows, pos % page] = k[:T]
        assert got is None
    else:
        f, axis = _freqs((rot,))
        y, both = _rope_64(k[:T], pos[:, None], rot, layout == "half", f, axis, 1.0, False)
        here = kv.k[1, rows, pos % page]
        assert ((here.double() - y).abs() <= _rope_bound(y, both, dtype)).all()
        want_k[1, rows, pos % page] = here
        y, both = _rope_64(q[:T], pos[:, None], rot, layout == "half", f, axis, 1.0, False)
        assert got is out and ((out[:T].double() - y).abs() <= _rope_bound(y, both, dtype)).all()
        assert (out[T:] == 3).all()
        # the same tokens at given positions
        again = kv.append(1, k, v, _cu(new), q=q, rope=rope, positions=torch.cat([pos, pos[:pad]]).int())
        assert torch.equal(again[:T], out[:T])
    assert torch.equal(kv.k, want_k) and torch.equal(kv.v, want_v)


def test_append_leaves_places_without_a_page():
    """Bad page numbers and lengths below the chunk write nothing outside and nothing elsewhere."""
    kv = ops.PagedKV.empty(1, 4, 16, 1, 64, 3, 2)
    kv.k.zero_(), kv.v.zero_()
    kv.table.copy_(_i32([[7, -3], [1, 2], [3, -1]]))
    kv.lens.copy_(_i32([20, 2, 40]))  # out of the pool; shorter than the chunk; past the table
    ones = torch.ones(12, 1, 64, device=DEV, dtype=torch.bfloat16)
    kv.append(0, ones, ones, _i32([0, 4, 8, 12]))
    assert kv.k[0, 1].view(16, 64).sum(1).tolist() == [64.0, 64.0] + [0.0] * 14
    assert kv.k.sum() == 128 and kv.v.sum() == 128


# ------------------------------------------------------------------------------- attention
def _attend_64(q, k, v, n, causal, scale):
    """q [n, Hq, D], k, v [len, Hk, D] -> out, softmax-weighted |v|, the largest sum |q||k| scale."""
    g = q.shape[1] // k.shape[1]
    q, k, v = q.double(), k.double().repeat_interleave(g, 1), v.double().repeat_interleave(g, 1)
    x = torch.einsum("ihd,jhd->hij", q, k) * scale
    L = k.shape[0]
    if causal:
        i = torch.arange(n, device=DEV)[:, None]
        seen = torch.arange(L, device=DEV) <= L - n + i
        x = x.masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True) if L else x.new_zeros(x.shape[0], n, 1)
    p = torch.exp(x - top.clamp(min=-1e300))
    p = torch.where(torch.isinf(x), 0.0, p)
    s = p.sum(-1, keepdim=True)
    p = p / torch.where(s > 0, s, 1.0)
    size = (torch.einsum("ihd,jhd->hij", q.abs(), k.abs()) * scale).amax(-1) if L else x.new_zeros(x.shape[0], n)
    return torch.einsum("hij,jhd->ihd", p, v), torch.einsum("hij,jhd->ihd", p, v.abs()), size.t()[..., None]


def _attend_bound(o, a, size, L, D, dtype):
    """Half a step of the result.  Each probability is rounded to the type (u, relative) and off by
    what its exponent is off: D products summed in fp32 (D 2^-23 of sum |q||k| scale), its scaling and
    subtraction (2^-22 of the same), and ex2's own 2^-22; numerator and sum alike (twice).  Sums of L
    terms in fp32 are off by L 2^-23."""
    u = U[dtype]
    d = size * (D * 2.0 ** -23 + 2.0 ** -22) + 2.0 ** -22
    return u * o.abs() + a * (u + 2 * d + L * 2.0 ** -23) * (1 + 2 * u) + TINY[dtype]


def _case(new, had, Hq, Hk, D, page, dtype, seed, spare=3, width=None, sharp=1.0):
    """A cache whose free slots and pages hold NaNs, and q."""
    B = len(new)
    lens = [a + b for a, b in zip(new, had)]
    need = [-(-n // page) for n in lens]
    P = sum(need) + spare
    width = width or max(need + [1])
    order = list(range(P))
    random.Random(seed).shuffle(order)
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    g = _gen(seed)
    k = torch.full((P, page, Hk, D), math.nan, device=DEV, dtype=dtype)
    v = k.clone()
    ks, vs = [], []
    for b in range(B):
        kb = (torch.randn(lens[b], Hk, D, device=DEV, generator=g) * sharp).to(dtype)
        vb = torch.randn(lens[b], Hk, D, device=DEV, generator=g).to(dtype)
        i = torch.arange(lens[b], device=DEV)
        rows = _i32(table[b]).long()[i // page] if lens[b] else i
        k[rows, i % page], v[rows, i % page] = kb, vb
        ks.append(kb)
        vs.append(vb)
    q = torch.randn(sum(new), Hq, D, device=DEV, generator=g).to(dtype)
    return q, k, v, _i32(table), _i32(lens), ks, vs


def _check(out, q, ks, vs, new, causal, scale, dtype):
    at = 0
    for b, n in enumerate(new):
        if n:
            o, a, size = _attend_64(q[at:at + n], ks[b], vs[b], n, causal, scale)
            got = out[at:at + n].double()
            L, D = ks[b].shape[0], q.shape[2]
            bad = ~((got - o).abs() <= _attend_bound(o, a, size, L, D, dtype))
            assert not bad.any(), (b, bad.nonzero()[:3].tolist(), (got - o).abs().max().item())
        at += n


SHAPES = [
    # new, had, Hq, Hk, D, page
    ([1], [0], 1, 1, 128, 16),                                     # the very first token
    ([1], [2000], 12, 12, 128, 64),
    ([1] * 9, [0, 1, 15, 16, 17, 63, 64, 1000, 5000], 8, 2, 128, 16),
    ([1] * 5, [127, 128, 129, 300, 70], 12, 1, 64, 48),            # 12 rows of a group of 12
    ([1] * 3, [9, 700, 40], 16, 1, 128, 32),
    ([2, 1, 4, 0, 3], [100, 64, 0, 10, 2000], 8, 4, 64, 16),       # a few drafted tokens
    ([1] * 70, [37 * i % 900 for i in range(70)], 4, 4, 128, 16),  # more sequences than a warp
    ([128], [0], 2, 2, 128, 128),
    ([130], [1000], 3, 3, 128, 128),
    ([300, 0, 1, 77], [0, 50, 400, 129], 8, 2, 128, 16),
    ([257, 33], [255, 1], 6, 1, 64, 48),                           # a group that is no power of two
    ([700], [3000], 5, 5, 64, 256),
    ([1, 640, 5], [2000, 64, 0], 7, 7, 128, 64),
    ([20, 30, 40] * 20, [5, 200, 64] * 20, 4, 2, 64, 32),
    ([1, 1, 1], [5, 300, 1000], 40, 1, 128, 16),                   # one token of a group of 40
    # items of several segments whose two halves see different numbers of key tiles
    ([1537, 600, 900], [100, 300, 7], 16, 4, 64, 16),
    ([1100, 700], [3, 0], 12, 12, 128, 64),
    ([1500, 2000, 900, 700], [0, 0, 0, 0], 8, 1, 64, 32),
    # more items than the machine has SMs, of many lengths: whole ones dealt out by length
    ([0 if i % 7 == 0 else 1 + 41 * i % 131 for i in range(90)], [97 * i % 1300 for i in range(90)], 8, 4, 128, 16),
    ([300] * 40, [0] * 40, 4, 4, 64, 64),
    ([130, 1, 1, 2, 64] * 12, [0, 700, 3000, 128, 5] * 12, 12, 4, 128, 32),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attend(shape, causal, dtype):
    new, had, Hq, Hk, D, page = SHAPES[shape]
    q, k, v, table, lens, ks, vs = _case(new, had, Hq, Hk, D, page, dtype, shape)
    out = ops.paged_attention(q, k, v, table, lens, _cu(new), causal=causal, max_new=max(new))
    _check(out, q, ks, vs, new, causal, D ** -0.5, dtype)
    # the other kernel: without a bound on the new tokens that of many rows, with a false one that of few
    many = ops.paged_attention(q, k, v, table, lens, _cu(new), causal=causal)
    few = ops.paged_attention(q, k, v, table, lens, _cu(new), causal=causal, max_new=1)
    _check(many, q, ks, vs, new, causal, D ** -0.5, dtype)
    _check(few, q, ks, vs, new, causal, D ** -0.5, dtype)
    if all(n == 1 for n in new):
        assert torch.equal(ops.paged_attention(q, k, v, table, lens, causal=causal), out) or Hq // Hk > 16
    # the cut of the work does not depend on timing
    assert torch.equal(out, ops.paged_attention(q, k, v, table, lens, _cu(new), causal=causal, max_new=max(new)))


@pytest.mark.parametrize("max_new", [1, 400])
def test_attend_rows_that_see_nothing(max_new):
    """Lengths below the chunk: the first tokens lie before the cache's start; and an empty cache."""
    new = [400, 6, 3]
    q, k, v, table, _, ks, vs = _case(new, [0, 0, 0], 4, 2, 64, 16, torch.bfloat16, 11)
    lens = [150, 0, 2]
    cu = _cu(new)
    out = ops.paged_attention(q, k, v, table, _i32(lens), cu, max_new=max_new)
    assert (out[:250] == 0).all() and (out[400:406] == 0).all() and (out[406] == 0).all()
    _check(out[250:400], q[250:400], [ks[0][:150]], [vs[0][:150]], [150], True, 0.125, torch.bfloat16)
    _check(out[407:], q[407:], [ks[2][:2]], [vs[2][:2]], [2], True, 0.125, torch.bfloat16)
    out = ops.paged_attention(q, k, v, table, _i32(lens), cu, causal=False, max_new=max_new)
    assert (out[400:406] == 0).all()
    _check(out[:400], q[:400], [ks[0][:150]], [vs[0][:150]], [400], False, 0.125, torch.bfloat16)
    # values of keys that some rows see do not reach rows that see none
    bad = v.clone()
    bad[table[0, 0].long()] = math.inf
    out = ops.paged_attention(q, k, bad, table, _i32(lens), cu, max_new=max_new)
    assert (out[:250] == 0).all() and not out[250:400].isfinite().any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attend_masked_values_weigh_nothing(dtype, D):
    """The largest values of the type behind the mask: the rows before them are the same to the bit."""
    new, had = [200, 70], [300, 0]
    q, k, v, table, lens, ks, vs = _case(new, had, 4, 2, D, 32, dtype, 27)
    for max_new in (1, 200):
        want = ops.paged_attention(q, k, v, table, lens, _cu(new), max_new=max_new)
        loud = v.clone()
        for b, (n, h) in enumerate(zip(new, had)):
            i = torch.arange(h + n // 2, h + n, device=DEV)
            loud[table[b].long()[i // 32], i % 32] = torch.finfo(dtype).max
        got = ops.paged_attention(q, k, loud, table, lens, _cu(new), max_new=max_new)
        for at, n in ((0, 200), (200, 70)):
            assert torch.equal(got[at:at + n // 2], want[at:at + n // 2])


@pytest.mark.parametrize("max_new", [1, 64])
def test_attend_sharp_scores(max_new):
    """Scores of hundreds, maxima that rise along the keys: the running maximum is moved many times."""
    new, had = [64, 1], [2000, 777]
    q, k, v, table, lens, ks, vs = _case(new, had, 4, 4, 128, 64, torch.bfloat16, 13, sharp=6.0)
    ramp = torch.linspace(0.1, 4, 2064, device=DEV)[:, None, None]
    i = torch.arange(2064, device=DEV)
    ks[0] = (ks[0] * ramp).bfloat16()
    k[table[0].long()[i // 64], i % 64] = ks[0]
    out = ops.paged_attention(q, k, v, table, lens, _cu(new), max_new=max_new, sm_scale=0.25)
    _check(out, q, ks, vs, new, True, 0.25, torch.bfloat16)


@pytest.mark.parametrize("max_new", [1, 90])
def test_attend_layouts(max_new):
    """q a slice of a projection, pages with heads outside tokens, k and v interleaved, out a slice."""
    new, had = [90, 3], [200, 31]
    q, k, v, table, lens, ks, vs = _case(new, had, 6, 2, 64, 32, torch.float16, 17)
    want = ops.paged_attention(q, k, v, table, lens, _cu(new), max_new=max_new)
    P, page, Hk, D = k.shape
    hnd = torch.empty(P, 2, Hk, page, D, device=DEV, dtype=k.dtype)
    hnd[:, 0], hnd[:, 1] = k.transpose(1, 2), v.transpose(1, 2)
    fused = torch.randn(93, 6 + 4, D, device=DEV).half()
    fused[:, 2:8] = q
    wide = torch.full((97, 6, 2 * D), 5.0, device=DEV, dtype=torch.float16)
    got = ops.paged_attention(fused[:, 2:8], hnd[:, 0].transpose(1, 2), hnd[:, 1].transpose(1, 2), table, lens,
                              _cu(new), max_new=max_new, out=wide[:93, :, D:])
    assert torch.equal(got, want)
    # tokens behind the last sequence: their rows stay
    qpad = torch.cat([q, q[:4]])
    wide.fill_(5.0)
    ops.paged_attention(qpad, k, v, table, lens, _cu(new), max_new=max_new, out=wide[..., :D])
    assert torch.equal(wide[:93, :, :D], want) and (wide[93:] == 5).all() and (wide[..., D:] == 5).all()
    # one query for all heads and tokens, without a copy of its own
    flat = q[:1, :1].expand(93, 6, D)
    assert torch.equal(ops.paged_attention(flat, k, v, table, lens, _cu(new), max_new=max_new),
                       ops.paged_attention(flat.contiguous(), k, v, table, lens, _cu(new), max_new=max_new))
    # an unaligned q is copied
    odd = torch.randn(93 * 6 * D + 1, device=DEV).half()
    odd[1:] = q.reshape(-1)
    assert torch.equal(ops.paged_attention(odd[1:].view(93, 6, D), k, v, table, lens, _cu(new), max_new=max_new), want)


@pytest.mark.parametrize("max_new", [1, 200])
def test_attend_bad_pages(max_new):
    """Page numbers outside the pool read as zeros; lengths past the table stop at its end."""
    new = [200, 1]
    q, k, v, table, lens, ks, vs = _case(new, [56, 99], 2, 2, 128, 32, torch.bfloat16, 19)
    table[0, 2], table[0, 5], table[1, 1] = 1 << 30, -7, k.shape[0]
    ks[0][64:96], vs[0][64:96], ks[0][160:192], vs[0][160:192] = 0, 0, 0, 0
    ks[1][32:64], vs[1][32:64] = 0, 0
    out = ops.paged_attention(q, k, v, table, lens, _cu(new), max_new=max_new)
    _check(out, q, ks, vs, new, True, 128 ** -0.5, torch.bfloat16)
    short = table[:, :4].contiguous()
    out = ops.paged_attention(q, k, v, short, lens, _cu(new), max_new=max_new, causal=False)
    _check(out, q, [x[:128] for x in ks], [x[:128] for x in vs], new, False, 128 ** -0.5, torch.bfloat16)


def test_attend_far_pages():
    """Offsets past 2^31 elements: the last pages of a pool of 2.2 G."""
    H, D, page, P = 8, 128, 64, 33600
    kv = ops.PagedKV.empty(1, P, page, H, D, 2, 40)
    assert kv.k.numel() > 2 ** 31 + 10 ** 7
    pages = list(range(P - 40, P))
    random.Random(3).shuffle(pages)
    kv.table.copy_(_i32([pages[:20] + [-1] * 20, pages[20:] + [-1] * 20]))
    kv.lens.copy_(_i32([1100, 1280]))
    g = _gen(21)
    new = [300, 5]
    k, v = (torch.randn(2380, H, D, device=DEV, generator=g).bfloat16() for _ in range(2))
    cu = _i32([0, 1100, 2380])
    kv.append(0, k, v, cu)
    q = torch.randn(305, H, D, device=DEV, generator=g).bfloat16()
    for max_new in (300, 1):
        out = kv.attend(0, q, _cu(new), max_new=max_new)
        _check(out, q, [k[:1100], k[1100:]], [v[:1100], v[1100:]], new, True, D ** -0.5, torch.bfloat16)


def test_attend_captured():
    """One graph over growing lengths: room, append, attention; replayed on another stream too."""
    H, D, page, B = 4, 64, 16, 3
    rope = ops.Rope(D, layout="half")
    one = _i32([1, 1, 1])
    cu = _i32([0, 1, 2, 3])
    x = torch.zeros(B, 3 * H, D, device=DEV, dtype=torch.bfloat16)
    kvs = [ops.PagedKV.empty(1, 40, page, H, D, B, 10) for _ in range(2)]
    for kv in kvs:
        kv.reserve(_i32([14, 0, 47]))
        kv.k.normal_(generator=_gen(23)), kv.v.normal_(generator=_gen(24))

    def step(kv):
        kv.reserve(one)
        q = kv.append(0, x[:, H:2 * H], x[:, 2 * H:], cu, q=x[:, :H], rope=rope)
        return kv.attend(0, q)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    spare = ops.PagedKV.empty(1, 40, page, H, D, B, 10)
    with torch.cuda.stream(side):
        step(spare)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(kvs[0])
    for i in range(20):
        x.copy_(torch.randn(x.shape, device=DEV, generator=_gen(30 + i)))
        if i % 2:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph.replay()
            torch.cuda.current_stream().wait_stream(side)
        else:
            graph.replay()
        want = step(kvs[1])
        assert torch.equal(y, want)
    assert kvs[0].lens.tolist() == [34, 20, 67]
    for a, b in zip((kvs[0].k, kvs[0].table, kvs[0].refs), (kvs[1].k, kvs[1].table, kvs[1].refs)):
        assert torch.equal(a, b)
    kvs[0].check()


def test_two_calls_at_once():
    """Calls on two streams do not share anything."""
    cases = [_case([1] * 8, [500 + 97 * i for i in range(8)], 8, 2, 128, 32, torch.bfloat16, 41),
             _case([300, 64], [1000, 77], 8, 2, 128, 32, torch.bfloat16, 42)]
    cus = [_cu([1] * 8), _cu([300, 64])]
    mx = [1, 300]
    want = [ops.paged_attention(*c[:5], cu, max_new=m) for c, cu, m in zip(cases, cus, mx)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for r in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i % 2, ops.paged_attention(*cases[i % 2][:5], cus[i % 2], max_new=mx[i % 2])))
    torch.cuda.synchronize()
    for i, y in got:
        assert torch.equal(y, want[i])


# ------------------------------------------------------------------------------- together
def test_streams_branch_and_go_on():
    """Two layers: prompts, single tokens, branches, dropped windows, a compaction; every chunk's
    attention against the tokens that the book says each stream has."""
    layers, Hq, Hk, D, page, seqs = 2, 6, 2, 64, 16, 6
    dt = torch.float16
    r = random.Random(5)
    kv = ops.PagedKV.empty(layers, 160, page, Hk, D, seqs, 40, dtype=dt)
    kv.k.fill_(math.nan), kv.v.fill_(math.nan)
    rope = ops.Rope(D, layout="interleaved", scaling="linear", factor=2.0)
    f = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D) / 2
    axis = torch.zeros(D // 2, dtype=torch.long, device=DEV)
    kept = [[[], []] for _ in range(seqs)]  # of each stream: k and v rows [layers, Hk, D]
    g = _gen(6)

    def chunk(new):
        T = sum(new)
        kv.reserve(_i32(new))
        at = [len(kept[b][0]) for b in range(seqs)]
        pos = torch.cat([torch.arange(a, a + n) for a, n in zip(at, new)]).to(DEV)
        rows = [[], []]
        for layer in range(layers):
            x = torch.randn(T, Hq + 2 * Hk, D, device=DEV, generator=g).to(dt)
            q, k, v = x.split((Hq, Hk, Hk), 1)
            q2 = kv.append(layer, k, v, _cu(new), q=q, rope=rope)
            y, both = _rope_64(k, pos[:, None], D, False, f, axis, 1.0, False)
            # what the cache holds is what attention is judged by; it is checked here once
            t0 = 0
            held = torch.empty_like(k)
            for b, n in enumerate(new):
                i = torch.arange(at[b], at[b] + n, device=DEV)
                held[t0:t0 + n] = kv.k[layer, kv.table[b].long()[i // page], i % page]
                t0 += n
            assert ((held.double() - y).abs() <= _rope_bound(y, both, dt)).all()
            rows[0].append(held), rows[1].append(v)
            ks = [torch.cat([torch.stack([t[layer] for t in kept[b][0]]) if kept[b][0] else k[:0],
                             held[sum(new[:b]):sum(new[:b + 1])]]) for b in range(seqs)]
            vs = [torch.cat([torch.stack([t[layer] for t in kept[b][1]]) if kept[b][1] else k[:0],
                             v[sum(new[:b]):sum(new[:b + 1])]]) for b in range(seqs)]
            out = kv.attend(layer, q2, _cu(new), max_new=max(new))
            _check(out, q2, ks, vs, new, True, D ** -0.5, dt)
        for i in range(2):
            both = torch.stack(rows[i], 1)
            t = 0
            for b, n in enumerate(new):
                kept[b][i] += list(both[t:t + n])
                t += n

    chunk([100, 33, 0, 0, 0, 0])
    chunk([1, 1, 0, 0, 0, 0])
    kv.fork(_i32([0, 1, 0]), _i32([2, 3, 5]))
    for a, d in ((0, 2), (1, 3), (0, 5)):
        kept[d] = [list(kept[a][0]), list(kept[a][1])]
    for _ in range(3):
        chunk([1, 1, 1, 1, 0, 1])
    chunk([40, 0, 17, 3, 50, 1])
    kv.release(_i32([0, 3]), _i32([2, 1]))  # windows that slide: the rotation of what stays does not
    for b, n in ((0, 2), (3, 1)):
        kept[b] = [kept[b][0][n * page:], kept[b][1][n * page:]]
    kv.release(_i32([5]))
    kept[5] = [[], []]
    kv.compact()
    used = int((kv.refs > 0).sum())
    assert (kv.refs[:used] > 0).all() and (kv.refs[used:] == 0).all()
    kv.fork(_i32([4]), _i32([5]))
    kept[5] = [list(kept[4][0]), list(kept[4][1])]
    for _ in range(2):
        chunk([r.randint(0, 5) for _ in range(seqs - 1)] + [1])
    chunk([64, 20, 1, 130, 2, 16])
    kv.check()


# ------------------------------------------------------------------------------- refusals
def test_refusals():
    bf = torch.bfloat16
    x = torch.zeros(4, 2, 64, device=DEV, dtype=bf)
    pos = torch.zeros(4, device=DEV, dtype=torch.int32)
    rope = ops.Rope(64)
    bad = [lambda: ops.fused_rope(x.double(), None, pos, rope),
           lambda: ops.fused_rope(x, x.float(), pos, rope),
           lambda: ops.fused_rope(x, x[:3], pos, rope),
           lambda: ops.fused_rope(x, None, pos[:3], rope),
           lambda: ops.fused_rope(x, None, pos.float(), rope),
           lambda: ops.fused_rope(x, None, pos, ops.Rope(66)),
           lambda: ops.fused_rope(x, None, pos, ops.Rope(64, axes=(32, 32))),
           lambda: ops.fused_rope(x, None, pos, rope, out_q=x.float()),
           lambda: ops.fused_rope(x, None, pos, rope, out_k=x),
           lambda: ops.fused_rope(x[0], None, pos, rope),
           lambda: ops.fused_rope(x, None, pos, ops.Rope(64, device="cpu")),
           lambda: ops.fused_rope(torch.zeros(1, 1, 300, device=DEV), None, pos[:1], rope),
           lambda: ops.fused_rope(x.float().requires_grad_(), None, pos, rope, out_q=x.float())]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    kv = ops.PagedKV.empty(1, 4, 16, 2, 64, 2, 3)
    cu = _i32([0, 2, 4])
    bad = [lambda: kv.append(0, x.half(), x, cu), lambda: kv.append(1, x, x, cu),
           lambda: kv.append(0, x, x[:3], cu), lambda: kv.append(0, x, x, cu[:2]),
           lambda: kv.append(0, x, x, cu.long()), lambda: kv.append(0, x, x, cu, q=x),
           lambda: kv.append(0, x, x, cu, positions=pos),
           lambda: kv.append(0, x, x, cu, rope=ops.Rope(64, axes=(32, 32))),
           lambda: kv.append(0, x, x, cu, rope=ops.Rope(128)), lambda: kv.append(0, x, x, cu, out_q=x),
           lambda: kv.reserve(_i32([1])), lambda: kv.reserve(torch.zeros(2, device=DEV)),
           lambda: kv.fork(_i32([0]), _i32([1, 1])), lambda: kv.fork(_i32([0] * 3), _i32([1] * 3)),
           lambda: kv.release(_i32([0]), _i32([1, 2])), lambda: kv.attend(-1, x, cu),
           lambda: kv.attend(0, x.half(), cu), lambda: kv.attend(0, x),
           lambda: kv.attend(0, x[:, :1].expand(4, 3, 64), cu), lambda: kv.attend(0, x, cu, max_new=0),
           lambda: kv.attend(0, x, cu, sm_scale=0.0), lambda: kv.attend(0, x, cu, sm_scale=-1.0),
           lambda: kv.attend(0, x, cu, sm_scale=math.inf), lambda: kv.attend(0, x, cu, out=x),
           lambda: kv.attend(0, x, cu, out=x.half()), lambda: kv.attend(0, x, cu[:2]),
           lambda: ops.PagedKV(kv.k, kv.v, kv.table, kv.lens[:1], kv.refs),
           lambda: ops.PagedKV(kv.k, kv.v, kv.table, kv.lens, kv.refs.long()),
           lambda: ops.PagedKV(kv.k, kv.v.half(), kv.table, kv.lens, kv.refs),
           lambda: ops.PagedKV(kv.k.float(), kv.v.float(), kv.table, kv.lens, kv.refs),
           lambda: ops.PagedKV(kv.k.transpose(2, 3), kv.v.transpose(2, 3), kv.table, kv.lens, kv.refs),
           lambda: ops.PagedKV.empty(1, 4, 24, 2, 64, 2), lambda: ops.PagedKV.empty(1, 4, 16, 2, 60, 2),
           lambda: ops.paged_attention(x, kv.k[0, :, :8], kv.v[0, :, :8], kv.table, kv.lens, cu),
           lambda: ops.paged_attention(x, kv.k[0].transpose(2, 3), kv.v[0].transpose(2, 3), kv.table, kv.lens, cu)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    for obj, name in ((kv, "table"), (kv, "k"), (kv, "status"), (rope, "freq")):
        with pytest.raises(AttributeError):
            setattr(obj, name, None)
    wide = ops.PagedKV.empty(1, 4, 16, 2, 72, 2, 3)
    with pytest.raises(NotImplementedError):
        wide.attend(0, torch.zeros(4, 2, 72, device=DEV, dtype=bf), cu)
    # nothing to do
    z = x[:0]
    assert kv.attend(0, z, _i32([0, 0, 0])).shape == (0, 2, 64)
    kv.append(0, z, z, _i32([0, 0, 0]))
    kv.check()
