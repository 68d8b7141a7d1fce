"""Which arrays an eviction takes for overlapping (no GPU: a call whose arrays
are good goes on to find that the pointers are none of the device's)."""

import pytest

from test_cache_attn_args import S, _lib, _shape, evict

SLOT = 2 * 2 * 128 * 64  # bytes of one cache slot of the shape: 2 KV heads, 128 positions, 64 values


def overlaps(**kw):
    assert evict(**kw) == 1
    return "overlap" in _lib()[1].lfm_ops_error().decode()


K, V, ACC, POS = S, 2 * S, 3 * S, 4 * S


@pytest.mark.parametrize("src,dst,stride,expected", [
    # K and V of a slot side by side, in place and from one such array to another
    ((K, K + SLOT), (K, K + SLOT), 32768, False),
    ((K, K + SLOT), (V, V + SLOT), 32768, False),
    # sources and destinations of a slot all side by side
    ((K, K + SLOT), (K + 2 * SLOT, K + 3 * SLOT), 65536, False),
    # with a gap, and V in front of K
    ((K + SLOT + 64, K), (K + SLOT + 64, K), 32768 + 64, False),
    # V begins inside K's slot, or reaches into the next slot's K
    ((K, K + SLOT - 16), (K, K + SLOT - 16), 32768, True),
    ((K, K + SLOT + 16), (K, K + SLOT + 16), 32768, True),
    ((K, K + SLOT), (V, V + SLOT - 16), 32768, True),
    # the destination's slots are the source's, one further
    ((K, V), (K + 2 * SLOT, 9 * S // 2), 16384, True),
    # behind the last slot
    ((K, V), (K + 4 * SLOT, V + 4 * SLOT), 16384, False),
    ((K, V), (K + 4 * SLOT - 16, V + 4 * SLOT), 16384, True),
])
def test_slots_that_lie_between_one_another(src, dst, stride, expected):
    in_place = src == dst
    assert overlaps(src=(*src, ACC, POS), dst=(*dst, ACC, POS) if in_place else (*dst, 7 * S, 8 * S), slot=stride) == expected


def test_a_record_between_the_slots():
    """lens_out in the gap between two slots is outside both; one element into a slot is not."""
    assert not overlaps(out=5 * S + SLOT, slot=16384 + 64)
    assert overlaps(out=5 * S + SLOT - 4, slot=16384 + 64)


def test_sizes_that_pass_64_bits_wrap_nowhere():
    """2^31 - 1 slots 2^40 values apart, or so large a record: their ends are not taken modulo 2^64."""
    sh = _shape(kv_heads=1024, heads=1024, ctx=1 << 24)
    assert overlaps(sh=sh, slots=0x7fffffff, slot=1 << 40, most=128)
    assert overlaps(slots=0x7fffffff, slot=1 << 40, src=(K, V, 1 << 62, POS), dst=(5 * S, 6 * S, 7 * S, 1 << 62))
