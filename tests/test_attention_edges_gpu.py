"""The paged cache, attention over it and rotary positions where a call could go wrong without an error:
refused room, streams that slide, values that are not finite, outputs that overlap, gradients."""
import pytest
import torch

import flashvsr_sm89_ops_b200 as ops
from flashvsr_sm89_ops_b200 import _lib
from test_attention_pages_gpu import _fill, _freqs, _gen, _i32, _rope_64, _rope_bound, _tokens

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
