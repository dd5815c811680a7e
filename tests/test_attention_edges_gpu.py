"""The paged cache, attention over it and rotary positions where a call could go wrong without an error:
refused room, streams that slide, values that are not finite, outputs that overlap, gradients."""
import copy
import math
import random

import pytest
import torch

import flashvsr_sm89_ops_b200 as ops
from flashvsr_sm89_ops_b200 import _lib
from test_attention_pages_gpu import U, _attend_64, _case, _check, _cu, _fill, _freqs, _gen, _i32, _rope_64, _rope_bound, _tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def no_timeouts():
    yield
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


# ------------------------------------------------------------------------------- refused room
def _chunk(T, H, D, seed, dtype=torch.bfloat16):
    g = _gen(seed)
    return tuple(torch.randn(T, H, D, device=DEV, generator=g).to(dtype) for _ in range(3))


@pytest.mark.parametrize("why,more,what", [("pages", [20, 3, 20, 0], "no free pages"),
                                           ("width", [20, 3, 70, 0], "table row"),
                                           ("arguments", [20, 3, -1, 0], "bad arguments")])
def test_append_behind_a_refused_reserve_writes_nothing(why, more, what):
    """Cached tokens, a branch's shared pages among them, stay to the bit until there is room."""
    H, D, page = 2, 64, 16
    kv = ops.PagedKV.empty(2, 7, page, H, D, 4, 5)
    _fill(kv, 50)
    rope = ops.Rope(D)
    kv.reserve(_i32([32, 20, 0, 0]))
    q, k, v = _chunk(52, H, D, 51)
    for layer in range(2):
        kv.append(layer, k, v, _i32([0, 32, 52, 52, 52]), rope=rope)
    kv.fork(_i32([0]), _i32([2]))  # two full pages, shared
    kv.check()
    was = [t.clone() for t in (kv.k, kv.v, kv.table, kv.lens, kv.refs)]
    cu = _i32([0, 20, 23, 43, 43])
    q, k, v = _chunk(43, H, D, 52)
    for again in range(2):  # the second time without a reserve of its own
        if not again:
            kv.reserve(_i32(more))
        for layer in range(2):
            q2 = q.clone()
            kv.append(layer, k, v, cu, q=q2, rope=rope, out_q=q2)
            assert torch.equal(q2, q)  # not rotated either: the step can be done again
        for t, w in zip((kv.k, kv.v, kv.table, kv.lens, kv.refs), was):
            assert torch.equal(t, w)
        with pytest.raises(RuntimeError, match="not appended" if again else what):
            kv.check()
    kv.release(_i32([1]))
    had = [_tokens(kv, b) for b in (0, 2)]
    kv.reserve(_i32([20, 3, 20, 0]))
    for layer in range(2):
        kv.append(layer, k, v, cu)
    kv.check()
    for b, (hk, hv), t0 in ((0, had[0], 0), (2, had[1], 23)):
        k2, v2 = _tokens(kv, b)
        assert torch.equal(k2[:, :32], hk) and torch.equal(v2[:, :32], hv)
        for layer in range(2):
            assert torch.equal(k2[layer, 32:], k[t0:t0 + 20]) and torch.equal(v2[layer, 32:], v[t0:t0 + 20])


def test_captured_step_runs_into_a_full_pool():
    """Replays past the last free page leave what is cached alone, and go on once there is room."""
    H, D, page = 1, 64, 16
    kv = ops.PagedKV.empty(1, 3, page, H, D, 2, 3)
    one, cu = _i32([1, 1]), _i32([0, 1, 2])
    x = torch.zeros(2, H, D, device=DEV, dtype=torch.bfloat16)
    kv.reserve(_i32([15, 16])), kv.append(0, *_chunk(31, H, D, 1)[:2], _i32([0, 15, 31]))
    kv.check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    spare = ops.PagedKV.empty(1, 3, page, H, D, 2, 3)
    with torch.cuda.stream(side):
        spare.reserve(one), spare.append(0, x, x, cu)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv.reserve(one)
        kv.append(0, x, x, cu)
    x.fill_(1.0)
    graph.replay()  # 16 and 17 tokens: the last page goes to the second stream
    kv.check()
    was = [t.clone() for t in (kv.k, kv.v, kv.lens, kv.refs)]
    for i in range(3):
        x.fill_(2.0 + i)
        graph.replay()
        assert all(torch.equal(t, w) for t, w in zip((kv.k, kv.v, kv.lens, kv.refs), was))
    with pytest.raises(RuntimeError, match="no free pages"):
        kv.check()
    kv.release(_i32([1]))
    x.fill_(9.0)
    graph.replay()
    kv.check()
    assert kv.lens.tolist() == [17, 1] and (_tokens(kv, 0)[0][0, 16:] == 9).all() and (_tokens(kv, 1)[0] == 9).all()


def test_append_leaves_shared_pages_alone():
    """A page of several sequences is not written to, whatever lens say: each keeps what it has."""
    H, D, page = 1, 64, 16
    kv = ops.PagedKV.empty(1, 8, page, H, D, 3, 4)
    _fill(kv, 3)
    kv.reserve(_i32([32, 16, 0]))
    kv.append(0, *_chunk(48, H, D, 4)[:2], _i32([0, 32, 48, 48]))
    kv.fork(_i32([0]), _i32([2]))
    kv.check()
    want_k, want_v = kv.k.clone(), kv.v.clone()
    q, k, v = _chunk(24, H, D, 5)
    oq = kv.append(0, k, v, _i32([0, 8, 16, 24]), q=q, rope=ops.Rope(D))  # nobody reserved anything
    with pytest.raises(RuntimeError, match="not appended"):
        kv.check()
    p = kv.table[1, 0].long()  # the middle stream's page is its own
    want_k[0, p, 8:], want_v[0, p, 8:] = kv.k[0, p, 8:], v[8:16]
    assert torch.equal(kv.k, want_k) and torch.equal(kv.v, want_v)
    f, axis = _freqs((D,))
    pos = torch.cat([torch.arange(24, 32), torch.arange(8, 16), torch.arange(24, 32)]).to(DEV)
    y, both = _rope_64(q, pos[:, None], D, False, f, axis, 1.0, False)
    assert ((oq.double() - y).abs() <= _rope_bound(y, both, q.dtype)).all()


# ------------------------------------------------------------------------------- streams that slide
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_positions_of_a_stream_that_slides(layout):
    """Default positions count every token that a stream ever had; branches go on where their parent is;
    a stream without tokens begins anew."""
    H, D, page, seqs = 2, 64, 16, 4
    dt = torch.float16
    kv = ops.PagedKV.empty(1, 60, page, H, D, seqs, 12, dtype=dt)
    rope = ops.Rope(D, layout=layout)
    f, axis = _freqs((D,))
    ever = [0] * seqs
    seed = 60

    def chunk(new):
        nonlocal seed
        seed += 1
        q, k, v = _chunk(sum(new), H, D, seed, dt)
        kv.reserve(_i32(new))
        oq = kv.append(0, k, v, _cu(new), q=q, rope=rope)
        pos = torch.cat([torch.arange(a, a + n) for a, n in zip(ever, new)]).to(DEV)
        y, both = _rope_64(q, pos[:, None], D, layout == "half", f, axis, 1.0, False)
        assert ((oq.double() - y).abs() <= _rope_bound(y, both, dt)).all()
        y, both = _rope_64(k, pos[:, None], D, layout == "half", f, axis, 1.0, False)
        t = 0
        for b, n in enumerate(new):
            if n:
                here = _tokens(kv, b)[0][0, -n:]
                assert ((here.double() - y[t:t + n]).abs() <= _rope_bound(y, both, dt)[t:t + n]).all()
            t += n
            ever[b] += n

    chunk([70, 40, 0, 5])
    kv.release(_i32([0, 1]), _i32([2, 1]))
    chunk([1, 1, 0, 1])
    chunk([20, 3, 0, 40])
    kv.release(_i32([3, 0]), _i32([0, 3]))
    kv.fork(_i32([0]), _i32([2]))
    ever[2] = ever[0]
    chunk([2, 2, 9, 1])
    assert kv.dropped.tolist() == [80, 16, 80, 0]
    kv.release(_i32([2]))             # all of it
    kv.release(_i32([1]), _i32([9]))  # more pages than it has
    ever[1] = ever[2] = 0
    assert kv.dropped.tolist() == [80, 0, 0, 0]
    chunk([1, 4, 3, 17])
    kv.compact()
    chunk([1, 1, 1, 1])
    kv.check()


def test_a_stream_that_slides_attends_as_one_that_does_not():
    """The same tokens with and without their oldest pages given back: attention of the next ones over what is
    kept is the same, as rotation goes by distance."""
    H, D, page = 2, 64, 16
    rope = ops.Rope(D)
    q, k, v = _chunk(100, H, D, 70, torch.float16)
    outs = []
    for slide in (False, True):
        kv = ops.PagedKV.empty(1, 10, page, H, D, 1, 10, dtype=torch.float16)
        kv.reserve(_i32([96])), kv.append(0, k[:96], v[:96], _i32([0, 96]), rope=rope)
        if slide:
            kv.release(_i32([0]), _i32([3]))
        kv.reserve(_i32([4]))
        q2 = kv.append(0, k[96:], v[96:], _i32([0, 4]), q=q[96:], rope=rope)
        if not slide:  # hide the first 48 keys by hand
            kv.table[0, :7] = kv.table[0, 3:].clone()
            kv.lens.sub_(48)
        outs.append(kv.attend(0, q2, _i32([0, 4])))
    assert torch.equal(*outs)


def test_streams_slide_branch_and_go_on():
    """Two layers: prompts, single tokens, branches, dropped windows, a compaction; every chunk's attention
    against the tokens that each stream has, rotated by their place among all that it ever had."""
    layers, Hq, Hk, D, page, seqs = 2, 6, 2, 64, 16, 6
    dt = torch.float16
    r = random.Random(5)
    kv = ops.PagedKV.empty(layers, 160, page, Hk, D, seqs, 40, dtype=dt)
    kv.k.fill_(math.nan), kv.v.fill_(math.nan)
    rope = ops.Rope(D, scaling="linear", factor=2.0)
    f, axis = _freqs((D,))
    f = f / 2
    held = [[torch.empty(layers, 0, Hk, D, device=DEV, dtype=dt)] * 2 for _ in range(seqs)]  # of each stream: k and v
    ever = [0] * seqs
    g = _gen(6)

    def chunk(new):
        kv.reserve(_i32(new))
        pos = torch.cat([torch.arange(a, a + n) for a, n in zip(ever, new)]).to(DEV)
        for b, n in enumerate(new):
            ever[b] += n
            held[b] = [torch.cat([t, t.new_zeros(layers, n, Hk, D)], 1) for t in held[b]]
        for layer in range(layers):
            x = torch.randn(sum(new), Hq + 2 * Hk, D, device=DEV, generator=g).to(dt)
            q, k, v = x.split((Hq, Hk, Hk), 1)
            q2 = kv.append(layer, k, v, _cu(new), q=q, rope=rope)
            for t, y in ((q, q2), (k, torch.cat([_tokens(kv, b)[0][layer, -n:] for b, n in enumerate(new) if n]))):
                want, both = _rope_64(t, pos[:, None], D, False, f, axis, 1.0, False)
                assert ((y.double() - want).abs() <= _rope_bound(want, both, dt)).all()
            t0 = 0
            for b, n in enumerate(new):
                if n:  # what the cache holds is what attention is judged by
                    held[b][0][layer, -n:] = _tokens(kv, b)[0][layer, -n:]
                    held[b][1][layer, -n:] = v[t0:t0 + n]
                t0 += n
            out = kv.attend(layer, q2, _cu(new), max_new=max(new))
            _check(out, q2, [h[0][layer] for h in held], [h[1][layer] for h in held], new, True, D ** -0.5, dt)

    def branch(src, dst):
        kv.fork(_i32(src), _i32(dst))
        for a, d in zip(src, dst):
            held[d], ever[d] = [t.clone() for t in held[a]], ever[a]

    def drop(b, n):
        kv.release(_i32([b]), None if n is None else _i32([n]))
        held[b] = [t[:, t.shape[1] if n is None else n * page:] for t in held[b]]
        if n is None:
            ever[b] = 0

    chunk([100, 33, 0, 0, 0, 0])
    chunk([1, 1, 0, 0, 0, 0])
    branch([0, 1, 0], [2, 3, 5])
    for _ in range(3):
        chunk([1, 1, 1, 1, 0, 1])
    chunk([40, 0, 17, 3, 50, 1])
    drop(0, 2), drop(3, 1)
    drop(5, None)
    kv.compact()
    used = int((kv.refs > 0).sum())
    assert (kv.refs[:used] > 0).all() and (kv.refs[used:] == 0).all()
    branch([0], [5])
    for _ in range(2):
        chunk([r.randint(0, 5) for _ in range(seqs - 1)] + [1])
    drop(5, 3)
    chunk([64, 20, 1, 130, 2, 16])
    kv.check()


def test_dropped_can_be_handed_in():
    D = 64
    rope = ops.Rope(D)
    kv = ops.PagedKV.empty(1, 4, 16, 1, D, 2, 2)
    far = torch.tensor([2 ** 33, 5], dtype=torch.int64, device=DEV)
    kv = ops.PagedKV(kv.k, kv.v, _i32([[0, 1], [2, 3]]), _i32([20, 3]), _i32([1] * 4), far)
    q, k, v = _chunk(5, 1, D, 80)
    got = kv.append(0, k, v, _i32([0, 2, 5]), q=q, rope=rope)
    pos = torch.tensor([2 ** 33 + 18, 2 ** 33 + 19, 5, 6, 7], device=DEV)
    assert torch.equal(got, ops.fused_rope(q, None, pos, rope)[0])
    for bad in (far.int(), far[:1], far.cpu(), far.view(2, 1)):
        with pytest.raises(ValueError):
            ops.PagedKV(kv.k, kv.v, kv.table, kv.lens, kv.refs, bad)


# ------------------------------------------------------------------------------- not finite
@pytest.mark.parametrize("max_new", [1, 300])
@pytest.mark.parametrize("D", [64, 128])
def test_nan_queries_reach_their_rows(D, max_new):
    """A head of a token that is NaN is NaN in the result, and the others are what they were."""
    new, had = [300, 1, 40], [700, 9000, 0]  # cut items and whole ones
    for dtype in (torch.bfloat16, torch.float16):
        q, k, v, table, lens, ks, vs = _case(new, had, 4, 2, D, 32, dtype, 90)
        want = ops.paged_attention(q, k, v, table, lens, _cu(new), max_new=max_new)
        rows = [(0, 1), (17, 0), (299, 3), (300, 2), (301, 0), (340, 1)]
        for t, h in rows:
            q[t, h, 5] = math.nan
        got = ops.paged_attention(q, k, v, table, lens, _cu(new), max_new=max_new)
        for t, h in rows:
            assert got[t, h].isnan().all(), (t, h)
            got[t, h] = want[t, h]
        assert torch.equal(got, want)


@pytest.mark.parametrize("max_new", [1, 200])
@pytest.mark.parametrize("bad", [math.nan, -math.inf])
def test_rows_whose_scores_are_not_finite(bad, max_new):
    """A row that sees keys, but has only NaN or -inf for scores, is NaN as its softmax is; 0 is for rows that see
    none.  And a stretch of NaN keys in a long cache is not lost between two parts of an item."""
    new, had = [200, 3], [0, 0]
    q, k, v, table, lens, ks, vs = _case(new, had, 2, 1, 64, 16, torch.bfloat16, 91)
    q = q.abs() + 0.5
    broken = k.clone()
    broken[table[1, 0].long(), :3] = bad  # all keys of the second sequence
    broken[table[0, 0].long(), 0] = bad   # and the only one of the first row
    out = ops.paged_attention(q, broken, v, table, lens, _cu(new), max_new=max_new)
    assert out[200:].isnan().all() and out[0].isnan().all()
    if bad == -math.inf:  # a weight of exactly nothing in the others
        x = ks[0].clone()
        x[0] = bad
        o, a, size = _attend_64(q[1:200], x, vs[0], 199, True, 0.125)
        assert out[1:200].isfinite().all() and (out[1:200].double() - o).abs().max() <= 2 * 2.0 ** -8 * 2 * a.max()
    none = ops.paged_attention(q, broken, v, table, _i32([0, 2]), _cu(new), max_new=max_new)
    assert (none[:200] == 0).all() and (none[200] == 0).all() and none[201:].isnan().all()
    q, k, v, table, lens, ks, vs = _case([1], [40000], 2, 1, 64, 16, torch.bfloat16, 92)
    k[table[0, 500:900].long()] = math.nan
    assert ops.paged_attention(q, k, v, table, lens, _cu([1]), max_new=max_new).isnan().all()


@pytest.mark.parametrize("max_new,shift", [(1, 15), (130, 7)])
@pytest.mark.parametrize("L", [40, 3000, 60000])
def test_many_small_weights_in_fp16(L, max_new, shift):
    """One key outweighs each of the others by 2^25: together they count all the same.  Weights are held as
    fp16 times 2^shift, so one is off by 2^-11 of itself or 2^-25-shift, whichever is more."""
    n, D = 2, 64
    kv = ops.PagedKV.empty(1, -(-L // 16) + 1, 16, 1, D, 1, dtype=torch.float16)
    kv.reserve(_i32([L]))
    k = torch.zeros(L, 1, D, device=DEV, dtype=torch.float16)
    g = _gen(93)
    k[:, 0, 0] = -17.5 + torch.rand(L, device=DEV, generator=g) * 0.1
    k[L // 3, 0, 0] = 0
    v = torch.rand(L, 1, D, device=DEV, generator=g).half() + 0.5
    v[L // 3] = 0
    kv.append(0, k, v, _i32([0, L]))
    q = torch.zeros(n, 1, D, device=DEV, dtype=torch.float16)
    q[:, :, 0] = 1
    out = kv.attend(0, q, _i32([0, n]), sm_scale=1.0, max_new=max_new, causal=False).double()
    want, a, _ = _attend_64(q, k, v, n, False, 1.0)
    # the exponent of each weight: 17.5 log2 e in fp32 and its subtraction, 2^-18; then as in _attend_bound
    tol = want * (2 * U[torch.float16] + 2.0 ** -18 + L * 2.0 ** -23) + L * 1.5 * 2.0 ** (-25 - shift) + 2.0 ** -25
    assert ((out - want).abs() <= tol).all(), ((out - want).abs() / tol).max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("max_new", [1, 200])
def test_scores_of_any_size(max_new, dtype):
    """Two kinds of keys, one score S for the one and -S for the other: the result is the mean of the first
    kind's values, whatever S is, though fp32 holds log2 e S to no better than 1 from 2^24 on."""
    n, L, D = 3, 900, 64
    g = _gen(103)
    kv = ops.PagedKV.empty(1, 60, 16, 1, D, 1, dtype=dtype)
    kv.reserve(_i32([L]))
    v = torch.randn(L, 1, D, device=DEV, generator=g).to(dtype)
    up = torch.rand(L, device=DEV, generator=g) < 0.3
    want = v[up].double().mean(0)
    # P in 16 bits (all of one value, so that is in the numerator alone), the sums, the output
    tol = v[up].double().abs().mean(0) * (U[dtype] + 2 * L * 2.0 ** -23) + U[dtype] * want.abs() + 2.0 ** -25
    for e in (*range(8, 15), *((20, 30, 50) if dtype == torch.bfloat16 else ())):
        for m in (1.0, 1.1, 1.3, 1.7, 1.9):
            k = torch.zeros(L, 1, D, device=DEV, dtype=dtype)
            k[:, 0, 0] = torch.where(up, m * 2.0 ** e, -m * 2.0 ** e)
            kv.append(0, k, v, _i32([0, L]))
            q = torch.zeros(n, 1, D, device=DEV, dtype=dtype)
            q[:, :, 0] = 2.0 ** e
            out = kv.attend(0, q, _i32([0, n]), sm_scale=1.0, max_new=max_new, causal=False).double()
            assert ((out - want).abs() <= tol).all(), (e, m, out[0, 0, :4])


@pytest.mark.parametrize("max_new", [1 << 58, 1 << 59, (1 << 63) - 1])
def test_huge_bounds_on_the_new_tokens(max_new):
    """max_new only picks the kernel: one that no product of it fits is that of many rows."""
    new, had = [3, 1], [50, 200]
    q, k, v, table, lens, ks, vs = _case(new, had, 64, 2, 64, 16, torch.bfloat16, 102)
    want = ops.paged_attention(q, k, v, table, lens, _cu(new), max_new=4)
    assert torch.equal(ops.paged_attention(q, k, v, table, lens, _cu(new), max_new=max_new), want)
    _check(want, q, ks, vs, new, True, 0.125, torch.bfloat16)


# ------------------------------------------------------------------------------- refusals
def test_outputs_that_overlap_are_refused():
    bf = torch.bfloat16
    x = torch.randn(8, 10, 64, device=DEV, generator=_gen(94)).to(bf)
    q, k, free = x[:, :4], x[:, 4:6], x[:, 6:]
    pos = torch.arange(8, device=DEV)
    rope = ops.Rope(64)
    one = torch.empty(1, 4, 64, device=DEV, dtype=bf)
    flat = x.view(-1)
    shifted = flat.as_strided((8, 4, 64), (640, 64, 1), 64)
    other = flat.as_strided((8, 4, 64), (256, 64, 1), 0)
    twice = torch.empty(8, 4, 64, device=DEV, dtype=bf)
    was = x.clone()
    for kw in ({"out_q": one.expand(8, 4, 64)}, {"out_q": twice[:, :1].expand(8, 4, 64)}, {"out_q": shifted},
               {"out_q": other}, {"out_q": k.repeat_interleave(2, 1), "out_k": k[:, :1].expand(8, 2, 64)},
               {"out_q": free, "out_k": free[:, 1:3]}, {"out_k": q[:, :2]}, {"out_q": x[:, 2:6]},
               {"out_q": twice.as_strided((8, 4, 64), (64, 64, 1))}):
        with pytest.raises(ValueError):
            ops.fused_rope(q, k, pos, rope, **kw)
            pytest.fail(str(kw.keys()))
    assert torch.equal(x, was)
    # what does not overlap is taken, in the same storage too
    want_q, want_k = ops.fused_rope(q, k, pos, rope)
    oq, ok = ops.fused_rope(q, k, pos, rope, out_q=free, out_k=k)
    assert torch.equal(oq, want_q) and torch.equal(ok, want_k) and torch.equal(x[:, :4], was[:, :4])
    halves = torch.zeros(8, 4, 128, device=DEV, dtype=bf)
    halves[..., :64] = q
    oq, _ = ops.fused_rope(halves[..., :64], None, pos, rope, out_q=halves[..., 64:])
    assert torch.equal(oq, want_q) and torch.equal(halves[..., :64], q)

    new = [5, 3]
    kv = ops.PagedKV.empty(1, 4, 16, 2, 64, 2, 2)
    kv.reserve(_i32(new)), kv.append(0, k, k, _cu(new))
    q = was[:, :4]
    for out in (one.expand(8, 4, 64), twice[:, :1].expand(8, 4, 64), was.view(-1).as_strided((8, 4, 64), (640, 64, 1), 64),
                was[:, 2:6], kv.k.view(-1)[:2048].view(8, 4, 64), kv.v.view(-1)[2048:4096].view(8, 4, 64),
                twice.as_strided((8, 4, 64), (64, 64, 1))):
        with pytest.raises(ValueError):
            kv.attend(0, q, _cu(new), out=out)
        with pytest.raises(ValueError):
            ops.paged_attention(q, kv.k[0], kv.v[0], kv.table, kv.lens, _cu(new), out=out)
    want = kv.attend(0, q, _cu(new))
    assert torch.equal(kv.attend(0, q, _cu(new), out=was[:, 6:]), want)
    for out in (one.expand(8, 4, 64), was[:, 1:5], kv.k.view(-1)[:2048].view(8, 4, 64)):
        with pytest.raises(ValueError):
            kv.append(0, was[:, 4:6], was[:, 4:6], _cu(new), q=q, rope=rope, out_q=out)


def test_nothing_to_write():
    kv = ops.PagedKV.empty(1, 4, 16, 2, 64, 2, 2)
    z = torch.empty(0, 2, 64, device=DEV, dtype=torch.bfloat16)
    out = torch.empty_like(z)
    assert kv.attend(0, z, _i32([0, 0, 0]), out=out) is out
    assert ops.paged_attention(z, kv.k[0], kv.v[0], kv.table, kv.lens, _i32([0, 0, 0]), out=out) is out
    rope = ops.Rope(64)
    assert ops.fused_rope(z, z, _i32([]), rope, out_q=out, out_k=out)[0] is out


@pytest.mark.parametrize("scale", [1e-60, 2.0 ** -151])
def test_scales_that_fp32_does_not_hold(scale):
    q, k, v, table, lens, ks, vs = _case([130], [3], 2, 2, 64, 16, torch.bfloat16, 95)
    for m in (1, 130):
        with pytest.raises(ValueError):
            ops.paged_attention(q, k, v, table, lens, _cu([130]), sm_scale=scale, max_new=m)
        for small in (2.0 ** -120, 2.0 ** -140):
            out = ops.paged_attention(q, k, v, table, lens, _cu([130]), sm_scale=small, max_new=m)
            _check(out, q, ks, vs, [130], True, small, torch.bfloat16)


# ------------------------------------------------------------------------------- gradients
def test_rope_tangents():
    import torch.autograd.forward_ad as fwd
    g = _gen(96)
    q, k, tq, tk = (torch.randn(9, h, 32, device=DEV, generator=g) for h in (4, 2, 4, 2))
    pos = torch.arange(9, device=DEV)
    rope = ops.Rope(24, scaling="yarn", factor=2.0, original_len=512)
    for inverse in (False, True):
        wq, wk = ops.fused_rope(tq, tk, pos, rope, inverse=inverse)
        pq, pk = ops.fused_rope(q, k, pos, rope, inverse=inverse)
        with fwd.dual_level():
            oq, ok = (fwd.unpack_dual(x) for x in ops.fused_rope(fwd.make_dual(q, tq), fwd.make_dual(k, tk), pos, rope,
                                                                 inverse=inverse))
            assert torch.equal(oq.primal, pq) and torch.equal(ok.primal, pk)
            assert torch.equal(oq.tangent, wq) and torch.equal(ok.tangent, wk)
            oq, ok = (fwd.unpack_dual(x) for x in ops.fused_rope(q, fwd.make_dual(k, tk), pos, rope, inverse=inverse))
            assert oq.tangent is None or (oq.tangent == 0).all()
            assert torch.equal(ok.tangent, wk)
            y, none = ops.fused_rope(fwd.make_dual(q, tq), None, pos, rope, inverse=inverse)
            assert none is None and torch.equal(fwd.unpack_dual(y).tangent, wq)
            with pytest.raises(ValueError):
                ops.fused_rope(fwd.make_dual(q, tq), None, pos, rope, out_q=torch.empty_like(q))


def test_what_has_no_gradient_says_so():
    """Results are what they are without gradients; a backward pass through them raises."""
    import torch.autograd.forward_ad as fwd
    bf = torch.bfloat16
    new = [5, 3]
    kv = ops.PagedKV.empty(1, 4, 16, 2, 64, 2, 2)
    kv.reserve(_i32(new))
    x = torch.randn(8, 8, 64, device=DEV, generator=_gen(97)).to(bf)
    rope = ops.Rope(64)
    want_q = kv.append(0, x[:, 4:6], x[:, 6:], _cu(new), q=x[:, :4], rope=rope)
    want = kv.attend(0, want_q, _cu(new))
    w = x.clone().requires_grad_()
    y = w * 1
    q2 = kv.append(0, y[:, 4:6], y[:, 6:], _cu(new), q=y[:, :4], rope=rope)
    assert torch.equal(q2.detach(), want_q)
    with pytest.raises(RuntimeError, match="no gradient"):
        q2.sum().backward(retain_graph=True)
    wide = torch.zeros(8, 4, 128, device=DEV, dtype=bf)
    for out in (kv.attend(0, q2, _cu(new)), kv.attend(0, y[:, :4], _cu(new)), kv.attend(0, q2, _cu(new), out=wide[..., 64:]),
                ops.paged_attention(x[:, :4], (kv.k[0].clone().requires_grad_() * 1), kv.v[0], kv.table, kv.lens, _cu(new))):
        with pytest.raises(RuntimeError, match="no gradient"):
            out.float().sum().backward(retain_graph=True)
    assert torch.equal(wide[..., 64:].detach(), want) and w.grad is None
    with torch.no_grad():
        assert not kv.attend(0, q2, _cu(new)).requires_grad
    assert not kv.attend(0, x[:, :4], _cu(new)).requires_grad
    with fwd.dual_level():
        assert torch.equal(kv.attend(0, want_q, _cu(new)), want)
        with pytest.raises((RuntimeError, NotImplementedError)):
            kv.attend(0, fwd.make_dual(want_q, want_q.clone()), _cu(new))


# ------------------------------------------------------------------------------- copies of a handle
def test_copies_have_their_own_tensors():
    rope = ops.Rope(64, axes=(32, 32))
    x = torch.randn(4, 2, 64, device=DEV, generator=_gen(98)).bfloat16()
    pos = torch.arange(8, device=DEV).view(4, 2)
    want = ops.fused_rope(x, None, pos, rope)[0]
    twin = copy.deepcopy(rope)
    rope.freq.zero_()
    assert torch.equal(ops.fused_rope(x, None, pos, twin)[0], want)
    kv = ops.PagedKV.empty(2, 8, 16, 2, 64, 3, 4)
    kv.reserve(_i32([20, 3, 0]))
    kv.append(1, *_chunk(23, 2, 64, 99)[:2], _i32([0, 20, 23, 23]))
    q = _chunk(23, 4, 64, 100)[0]
    want = kv.attend(1, q, _i32([0, 20, 23, 23]))
    kv.name = "mine"
    twin = copy.deepcopy(kv)
    assert twin.name == "mine" and twin.status.data_ptr() + 4 == twin.refused.data_ptr()
    assert not {t.data_ptr() for t in (twin.k, twin.v, twin.table, twin.lens, twin.refs, twin.dropped, twin.status, twin._ws)} \
        & {t.data_ptr() for t in (kv.k, kv.v, kv.table, kv.lens, kv.refs, kv.dropped, kv.status, kv._ws)}
    twin.release(_i32([0]))
    twin.reserve(_i32([0, 17, 4]))
    twin.append(1, *_chunk(21, 2, 64, 101)[:2], _i32([0, 0, 17, 21]))
    assert kv.lens.tolist() == [20, 3, 0] and kv.refs.tolist() == [1, 1, 1, 0, 0, 0, 0, 0]
    assert torch.equal(kv.attend(1, q, _i32([0, 20, 23, 23])), want)
    assert twin.lens.tolist() == [0, 20, 4]
    kv.check(), twin.check()


# ------------------------------------------------------------------------------- long lists
def test_lists_too_long_for_shared_memory():
    """More sequences, pages of one call and branches than the kernels keep in shared memory."""
    from test_attention_pages_gpu import Book
    seqs, page = 6000, 16
    r = random.Random(8)
    kv = ops.PagedKV.empty(1, 30000, page, 1, 8, seqs, 6, dtype=torch.float16)
    _fill(kv, 9)
    book = Book.of(kv)
    more = [r.choice((0, 5, 16, 40, 48)) if b % 2 else 0 for b in range(seqs)]
    assert sum(book.pages(n) for n in more) > 2048
    kv.reserve(_i32(more))
    book.reserve(more)
    book.check(kv)
    dst = [b for b in range(0, seqs, 2)]
    r.shuffle(dst)
    dst = dst[:2500]
    src = [r.randrange(1, seqs, 2) for _ in dst]
    some = r.sample(range(len(dst)), 40)
    before = [_tokens(kv, src[i]) for i in some]
    kv.fork(_i32(src), _i32(dst))
    book.fork(src, dst)
    book.check(kv)
    for i, (k, v) in zip(some, before):
        k2, v2 = _tokens(kv, dst[i])
        assert torch.equal(k, k2) and torch.equal(v, v2)
    drop = r.sample(range(seqs), 3000)
    count = [r.choice((0, 1, 2, 100)) for _ in drop]
    kv.release(_i32(drop), _i32(count))
    book.release(drop, count)
    book.check(kv)
    kv.compact()
    book.compact()
    book.check(kv)
    more = [r.choice((0, 1, 20)) if n <= 40 else 0 for n in book.lens]
    kv.reserve(_i32(more))
    book.reserve(more)
    book.check(kv)
    kv.check()
