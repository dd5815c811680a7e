"""Host side of the paged cache and of rotary positions: what the C entry points and the handles refuse."""
from flashvsr_sm89_ops_b200 import _lib


def test_append_needs_a_place_for_its_refusal():
    args = (0, 0, 0, 0, 0, 0, 0, 16, 128, 64, 16, 128, 64, 2, 4, 64, 0, 0, 0, 0, 0, 1, 0, 0, 1.0, 16, 16, 16, 2, 2, 4, 16,
            16, 16, 2048)
    for kw in ({"refused": 16}, {"refs": 16}):
        assert _lib.load().fvb_kv_append(_lib.KV_APPEND_ARGS(*args, **kw), None) == _lib.FVB_ERR_INVALID
