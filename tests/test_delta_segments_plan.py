"""Which long sequences the gated delta rule cuts into segments, by the scratch that the library asks for (no GPU)."""
import ctypes

import pytest

from linrec_amd import _delta


def scratch(batch, time, heads, key_dim, value_dim, packed=0):
    a = _delta.Delta(dtype=2, key_heads=heads, heads=heads, key_dim=key_dim, value_dim=value_dim, batch=batch, time=time, sequences=packed or batch)
    if packed:
        a.cu_seqlens = 16  # (not read)
    return _delta._lib.linrec_delta_scratch_bytes(ctypes.byref(a), 0)


def segments(time, heads, key_dim, value_dim, batch=1):
    """How many a sequence has; 64 positions of a head take the same scratch in a call that is too short to be cut."""
    width, columns = 64 if key_dim <= 64 else 128 if key_dim <= 128 else 256, -(-value_dim // 32) * 32
    chunk = 2 * 4096 * 4 + 768
    more = scratch(batch, time, heads, key_dim, value_dim) - batch * -(-time // 64) * heads * chunk
    each = batch * heads * ((columns + width) * width + columns * width) * 4
    assert more >= 0 and more - more // each * each < 5 * 256
    return more // each


def test_sizes_that_are_cut_and_that_are_not():
    assert segments(512, 4, 128, 128) == 0 and segments(448, 1, 64, 64) == 0  # short
    assert segments(8192, 48, 128, 128) == 0 and segments(4096, 16, 128, 128, batch=8) == 0  # many heads
    assert segments(8192, 16, 128, 128) == 8 and segments(8192, 32, 128, 128) == 4
    # 11 chunks at once are 22 halves of a chunk's time, in two segments 2 * 6 * 2 + 6; 12 are 24, in three segments 2 * 4 * 2 + 7
    assert segments(704, 1, 64, 64) == 0 and segments(768, 1, 64, 64) == 3


@pytest.mark.parametrize("key_dim,value_dim", [(16, 8), (64, 64), (100, 72), (256, 300)])
@pytest.mark.parametrize("heads", [1, 3, 40, 300])
def test_segments_have_four_chunks_or_more_and_none_is_empty(heads, key_dim, value_dim):
    for time in (1, 64, 500, 513, 1700, 8191, 8192, 100001):
        n, chunks = segments(time, heads, key_dim, value_dim), -(-time // 64)
        assert n == 0 or 2 <= n <= chunks / 4
        assert n == 0 or -(-chunks // -(-chunks // n)) == n


def test_packed_sequences_have_room_for_every_segment():
    """Any lengths that add up to `time`: a sequence of c chunks has ceil(c / segment) of them."""
    time, sequences = 100001, 3
    need = scratch(1, time, 1, 64, 32, packed=sequences)
    slots = time // 64 + sequences
    each = ((32 + 64) * 64 + 32 * 64) * 4
    parts = (need - slots * (2 * 4096 * 4 + 768)) // each
    segment = min(s for s in range(1, slots) if slots // s + sequences <= parts)
    for lengths in ((time, 0, 0), (1, 1, time - 2), (33333, 33334, 33334), (64 * segment + 1, 64 * segment + 1, time - 128 * segment - 2)):
        assert sum(-(-(-(-n // 64)) // segment) for n in lengths) <= parts
