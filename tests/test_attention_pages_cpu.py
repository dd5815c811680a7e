"""Host side of the rotary and paged-cache operators: frequencies, refusals, C argument checks."""
import math

import pytest
import torch

import flashvsr_sm89_ops_b200 as ops
from flashvsr_sm89_ops_b200 import _lib


def _turns(rope):
    return [(t % 2 ** 64) / 2 ** 64 * 2 * math.pi for t in rope.freq.tolist()]


def test_frequencies():
    r = ops.Rope(128, device="cpu")
    for i, w in enumerate(_turns(r)):
        assert abs(w - 10000.0 ** (-2 * i / 128)) <= 2.0 ** -52 * w + 2.0 ** -61
    assert r.axis.tolist() == [0] * 64 and r.axes == 1 and r.scale == 1.0
    a = ops.Rope(128, axes=(44, 42, 42), device="cpu")
    assert a.axes == 3 and a.axis.tolist() == [0] * 22 + [1] * 21 + [2] * 21
    from flashvsr_sm89_ops_b200.wan_video_dit import precompute_freqs_cis_3d
    want = torch.cat([f[1].angle() for f in precompute_freqs_cis_3d(128)])
    assert torch.allclose(torch.tensor(_turns(a), dtype=torch.float64), want, rtol=0, atol=1e-14)


def test_scalings_meet_at_their_ends():
    plain = _turns(ops.Rope(64, device="cpu"))
    for s in ("linear", "ntk", "yarn"):
        same = ops.Rope(64, scaling=s, factor=1.0, original_len=2048, device="cpu")
        assert _turns(same) == pytest.approx(plain, rel=1e-13) and same.scale == 1.0
    # ntk keeps the fastest pair and slows the slowest by the factor
    n = _turns(ops.Rope(64, scaling="ntk", factor=8.0, device="cpu"))
    assert n[0] == pytest.approx(plain[0]) and n[-1] == pytest.approx(plain[-1] / 8)
    y = ops.Rope(64, scaling="yarn", factor=8.0, original_len=2048, device="cpu")
    t = _turns(y)
    assert t[0] == pytest.approx(plain[0]) and t[-1] == pytest.approx(plain[-1] / 8)
    assert all(p / 8 * (1 - 1e-12) <= x <= p * (1 + 1e-12) for x, p in zip(t, plain))
    assert y.scale == pytest.approx(0.1 * math.log(8) + 1)
    assert ops.Rope(64, scaling="yarn", factor=8.0, original_len=2048, attention_factor=1.0, device="cpu").scale == 1.0


@pytest.mark.parametrize("args,kw", [((7,), {}), ((-2,), {}), ((8,), {"layout": "other"}), ((8,), {"scaling": "other"}),
                                     ((8,), {"theta": 1.0}), ((8,), {"theta": math.inf}),
                                     ((8,), {"scaling": "linear", "factor": 0.5}),
                                     ((8,), {"scaling": "yarn", "factor": 2.0}), ((8,), {"axes": (4, 2)}),
                                     ((8,), {"axes": (5, 3)}), ((8,), {"axes": ()}),
                                     ((8,), {"scaling": "yarn", "factor": 2.0, "original_len": 64, "beta_fast": 1.0})])
def test_rope_refuses(args, kw):
    with pytest.raises(ValueError):
        ops.Rope(*args, device="cpu", **kw)


def test_host_tensors_are_refused():
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.fused_rope(x, None, i, ops.Rope(64, device="cpu"))
    with pytest.raises(ValueError, match="CUDA"):
        ops.PagedKV.empty(1, 4, 16, 2, 64, 2, device="cpu")
    p = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention(x, p, p, i.view(2, 1), i)


def test_c_arguments():
    """Each refused before anything is launched: no device is there."""
    lib = _lib.load()
    bad, unsupported = _lib.FVB_ERR_INVALID, _lib.FVB_ERR_UNSUPPORTED

    def rope(T=4, D=64, rot=64, dtype=0, Hq=2, Hk=0, axes=1, q=16, pos=16, freq=16, axis=16):
        return lib.fvb_rope(_lib.ROPE_ARGS(q, Hq * D, D, Hq, q, Hq * D, D, 0, 0, 0, Hk, 0, 0, 0, T, D, rot, 0, dtype,
                                           pos, 0, axes, freq, axis, 1.0, 0), None)

    for kw in ({"T": -1}, {"D": 257}, {"D": 0}, {"rot": 65}, {"rot": 66}, {"rot": -2}, {"dtype": 3}, {"Hq": 4097},
               {"Hk": 1}, {"axes": 0}, {"axes": 17}, {"q": 0}, {"pos": 0}, {"freq": 0},
               {"axes": 2, "axis": 0}):
        assert rope(**kw) == bad, kw
    assert rope(T=0) == _lib.FVB_OK
    assert lib.fvb_rope(None, None) == lib.fvb_kv_append(None, None) == lib.fvb_paged_attn(None, None) == bad

    def append(T=4, D=64, rot=0, dtype=0, Hk=2, B=2, page=16, pages=4, width=2, axes=1, k=16, cu=16, pool=16):
        return lib.fvb_kv_append(_lib.KV_APPEND_ARGS(0, 0, 0, 0, 0, 0, 0, k, Hk * D, D, k, Hk * D, D, Hk, T, D, rot, 0,
                                                     dtype, 0, 0, axes, 0, 0, 1.0, cu, 16, 16, B, width, pages, page,
                                                     pool, pool, page * Hk * D), None)

    for kw in ({"T": -1}, {"D": 300}, {"rot": 2}, {"dtype": 2}, {"Hk": 0}, {"page": 0}, {"pages": -1}, {"width": -1},
               {"axes": 2}, {"k": 0}, {"cu": 0}, {"pool": 0}, {"B": -1}):
        assert append(**kw) == bad, kw
    assert append(T=0) == _lib.FVB_OK

    def attn(T=4, B=4, Hq=2, Hk=2, D=64, page=16, pages=4, width=2, max_new=1, scale=0.1, dtype=0, q=16, ws=16, cu=0,
             stride=0):
        return lib.fvb_paged_attn(_lib.PAGED_ATTN_ARGS(q, Hq * D + stride, D, 16, 8, 8, 8, 16, 8, 8, 8, 16, width, 16,
                                                       cu, T, B, Hq, Hk, D, pages, page, max_new, 1, scale, dtype, 32,
                                                       Hq * D, D, ws), None)

    for kw in ({"Hk": 0}, {"Hq": 3}, {"Hq": 0}, {"page": 8}, {"page": 24}, {"page": 0}, {"pages": 0}, {"width": -1},
               {"width": 1 << 28}, {"max_new": 0}, {"scale": 0.0}, {"scale": -1.0}, {"scale": math.inf},
               {"scale": math.nan}, {"dtype": 2}, {"q": 0}, {"q": 24}, {"ws": 0}, {"T": 5}, {"B": -1},
               {"stride": 4}):
        assert attn(**kw) == bad, kw
    assert attn(D=96) == unsupported and attn(D=256) == unsupported
    assert attn(T=0) == _lib.FVB_OK and attn(B=0) == _lib.FVB_OK

    def pages(table=16, seqs=2, width=2, pages=4, page=16, k=16, layers=1, layer=1024, stride=256, row=16, ws=16):
        return _lib.PAGES(table, 16, 16, 16, seqs, width, pages, page, k, 16, layers, layer, stride, row, ws)

    fns = [lambda c: lib.fvb_pages_reserve(c, 16, None), lambda c: lib.fvb_pages_fork(c, 16, 16, 1, None),
           lambda c: lib.fvb_pages_release(c, 16, None, 1, None), lambda c: lib.fvb_pages_compact(c, None)]
    for fn in fns:
        assert fn(None) == bad
        for kw in ({"page": 0}, {"page": 1 << 24}, {"table": 0}, {"seqs": -1}, {"seqs": (1 << 17) + 1}, {"width": -1},
                   {"seqs": 1 << 17, "width": 1 << 14}, {"pages": -1}, {"ws": 0}, {"ws": 24}):
            assert fn(pages(**kw)) == bad, kw
    for fn in fns[1::2]:
        for kw in ({"k": 24}, {"k": 0}, {"layer": 8}, {"stride": 250}, {"row": 8}, {"row": 0}, {"layers": -1}):
            assert fn(pages(**kw)) == bad, kw
    assert lib.fvb_pages_reserve(pages(), None, None) == bad
    assert lib.fvb_pages_reserve(pages(seqs=0), 16, None) == _lib.FVB_OK
    assert lib.fvb_pages_fork(pages(), 16, 16, -1, None) == bad
    assert lib.fvb_pages_fork(pages(), 16, 16, 3, None) == bad  # more branches than sequences
    assert lib.fvb_pages_fork(pages(), 16, None, 1, None) == bad
    assert lib.fvb_pages_fork(pages(), 16, 16, 0, None) == _lib.FVB_OK
    assert lib.fvb_pages_release(pages(), None, None, 1, None) == bad
    assert lib.fvb_pages_release(pages(), 16, None, 0, None) == _lib.FVB_OK
    assert lib.fvb_pages_compact(pages(pages=0), None) == _lib.FVB_OK
    assert lib.fvb_pages_workspace_bytes(10, 100) >= 4 * (11 + 100)
    assert lib.fvb_paged_attn_workspace_bytes(1, 8, 2, 128) < lib.fvb_paged_attn_workspace_bytes(64, 8, 2, 128)
