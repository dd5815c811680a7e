"""Host side of the paged cache and of rotary positions: frequencies, what the C entry points and the handles refuse."""
import copy
import math
import pickle
import random

import pytest
import torch

import flashvsr_sm89_ops_b200 as ops
from flashvsr_sm89_ops_b200 import _lib
from flashvsr_sm89_ops_b200.paged_kv import _followed
from flashvsr_sm89_ops_b200.rope import _clash, _own


@pytest.mark.parametrize("d,original,theta", [(128, 131072, 10000.0), (128, 4096, 10000.0), (64, 32768, 500.0),
                                              (4, 4096, 10000.0), (6, 4096, 10000.0), (2, 4096, 10000.0),
                                              (96, 8, 10000.0), (80, 1 << 40, 10000.0)])
def test_yarn_by_its_definition(d, original, theta):
    """Pair i turns n = original theta^(-2i/d) / 2 pi times.  The pair (a real number) of n = 32 rounded down and
    that of n = 1 rounded up, both kept within the d channels, are the ends of the ramp."""
    s = 8.0
    rope = ops.Rope(d, theta=theta, scaling="yarn", factor=s, original_len=original, device="cpu")
    got = [(t % 2 ** 64) / 2 ** 64 * 2 * math.pi for t in rope.freq.tolist()]
    at = [d / 2 * math.log(original / (2 * math.pi * n)) / math.log(theta) for n in (32, 1)]
    low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), d - 1)
    for i, w in enumerate(got):
        plain = theta ** (-2 * i / d)
        turns = original * plain / (2 * math.pi)
        r = 0.0 if i <= low else 1.0 if i >= high else (i - low) / (high - low)
        assert w == pytest.approx(plain * (1 - r) + plain / s * r, rel=1e-12)
        if turns > 1 and at[1] <= d - 1:
            assert w > plain / s  # it turns in the original length: not stretched in full


def test_append_needs_a_place_for_its_refusal():
    args = (0, 0, 0, 0, 0, 0, 0, 16, 128, 64, 16, 128, 64, 2, 4, 64, 0, 0, 0, 0, 0, 1, 0, 0, 1.0, 16, 16, 16, 2, 2, 4, 16,
            16, 16, 2048)
    for kw in ({"refused": 16}, {"refs": 16}):
        assert _lib.load().fvb_kv_append(_lib.KV_APPEND_ARGS(*args, **kw), None) == _lib.FVB_ERR_INVALID


@pytest.mark.parametrize("max_new,Hq,Hk", [(1 << 59, 64, 2), (1 << 62, 16, 4), ((1 << 63) - 1, 8, 4), (17, 4, 4),
                                           (1, 17, 1), (9, 2, 1)])
def test_many_rows_however_large_their_bound(max_new, Hq, Hk):
    """The kernel for few rows takes tiles of 16 / (Hq / Hk) whole tokens: none at all for larger groups."""
    ws = _lib.load().fvb_paged_attn_workspace_bytes
    assert ws(max_new, Hq, Hk, 128) == ws(17, 1, 1, 128) > ws(16, 1, 1, 128)
    assert ws(16, 4, 4, 128) == ws(1, 16, 1, 128) == ws(8, 2, 1, 128) == ws(5, 3, 1, 128) == ws(16, 1, 1, 128)


def _attend(T=4, B=4, Hq=2, D=64, page=16, width=2, scale=0.1, q=16):
    return _lib.load().fvb_paged_attn(_lib.PAGED_ATTN_ARGS(q, Hq * D, D, 16, 8, 8, 8, 16, 8, 8, 8, 16, width, 16, 0, T, B,
                                                           Hq, Hq, D, 4, page, 1, 1, scale, 0, 32, Hq * D, D, 16), None)


@pytest.mark.parametrize("scale", [1e-60, 2.0 ** -151, 5e-324])
def test_scales_that_are_nothing_in_fp32(scale):
    assert _attend(scale=scale, T=0, B=0) == _lib.FVB_ERR_INVALID
    assert _attend(scale=2.0 ** -149, T=0, B=0) == _lib.FVB_OK


def test_tables_up_to_the_last_key():
    for page, width, rc in ((16, (1 << 27) - 1, _lib.FVB_ERR_INVALID), (1024, (1 << 21) - 1, _lib.FVB_OK),
                            (16, (1 << 27) - 63, _lib.FVB_ERR_INVALID), (16, (1 << 27) - 64, _lib.FVB_OK)):
        assert _attend(page=page, width=width, T=0, B=0) == rc, (page, width)


def _elements(rows, D):
    p, T, H, t, h, e = rows
    return {p // e + i * t + j * h + c for i in range(T) for j in range(H) for c in range(D)}


def test_rows_that_share_elements():
    """Against the sets themselves: nothing shared is missed, and of rows of equal strides nothing else refused."""
    r = random.Random(1)
    shared = apart = 0
    for _ in range(20000):
        D = r.choice((1, 2, 4))
        h = r.choice((D, D + 1, 2 * D, 3 * D, 40))
        t = r.choice((h, 3 * h, 4 * h + 1, 7 * D, 2))
        sets = []
        for _ in range(2):
            same = r.random() < 0.8
            sets.append((2 * r.randint(0, 60), r.randint(0, 4), r.randint(0, 3), t if same else r.choice((h, 5 * h, D)),
                         h if same else r.choice((D, t)), 2))
        a, b = sets
        want = bool(_elements(a, D) & _elements(b, D))
        got = _clash(a, b, D)
        assert got or not want, (a, b, D)
        if (a[3:5] == b[3:5]) and a[1] and b[1]:
            assert got == want, (a, b, D)
            shared += want
            apart += not want
        rows = _elements(a, D)
        if len(rows) < a[1] * a[2] * D:
            with pytest.raises(ValueError):
                _own(a, D, "out", "test")
    assert shared > 1000 and apart > 1000
    _own((0, 8, 4, 640, 64, 2), 64, "out", "test")
    _own((0, 8, 4, 64, 512, 2), 64, "out", "test")  # heads outside tokens
    _own((0, 8, 1, 64, 1, 2), 64, "out", "test")
    _own((0, 1, 4, 0, 64, 2), 64, "out", "test")


def test_results_that_autograd_follows():
    w = torch.randn(3, 4, requires_grad=True)
    x = w * 1
    for y in (torch.zeros(3, 4), torch.zeros(3, 8)[:, 4:], torch.zeros(4, 3, 4).unbind(0)[1], torch.zeros(3, 8).chunk(2, 1)[0]):
        z = _followed("this", y, None, x)
        assert z.data_ptr() == y.data_ptr() and z.stride() == y.stride()
        with pytest.raises(RuntimeError, match="this has no gradient"):
            z.sum().backward()
    for y in (x, w):  # an input as the result, a leaf too
        z = _followed("this", y, y)
        assert z.data_ptr() == y.data_ptr()
        with pytest.raises(RuntimeError, match="this has no gradient"):
            z.sum().backward()
    y = torch.zeros(3, 4)
    assert _followed("this", y, w.detach(), None) is y and not y.requires_grad
    with torch.no_grad():
        assert _followed("this", y, w) is y and not y.requires_grad


def test_copies_of_a_rope_have_their_own_tensors():
    rope = ops.Rope(64, axes=(32, 32), scaling="yarn", factor=2.0, original_len=512, device="cpu")
    for twin in (copy.deepcopy(rope), pickle.loads(pickle.dumps(rope)), copy.deepcopy({"a": [rope]})["a"][0]):
        assert twin._freq == twin.freq.data_ptr() != rope.freq.data_ptr()
        assert twin._axis == twin.axis.data_ptr() != rope.axis.data_ptr()
        assert torch.equal(twin.freq, rope.freq) and torch.equal(twin.axis, rope.axis) and repr(twin) == repr(rope)
    same = copy.copy(rope)
    assert same._freq == rope._freq == rope.freq.data_ptr()
