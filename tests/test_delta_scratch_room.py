"""Scratch of the gated delta rule has room for every chunk and segment that the kernels number, whatever cu_seqlens holds (no GPU).

The sizes are computed here from the rule that cuts sequences, written down again, and compared with the library's; the numbers of chunks and
segments are those that the kernels give them."""
import ctypes
import random

import pytest

from linrec_amd import _delta

CHUNK, CUS = 64, 256


def cdiv(a, b):
    return -(-a // b)


def sizes(batch, time, heads, key_dim, value_dim, packed):
    """(slots, segment, parts, width, columns) of a call; `packed`: sequences, or 0."""
    width, columns = 64 if key_dim <= 64 else 128 if key_dim <= 128 else 256, cdiv(value_dim, 32) * 32
    of_block = 16 * (4 if columns > 32 else 2)
    blocks, sequences = cdiv(columns, of_block), packed or batch
    slots = time // CHUNK + sequences if packed else batch * cdiv(time, CHUNK)
    one, both, chunks = sequences * heads * blocks, sequences * heads * (blocks + width // of_block), cdiv(slots, sequences)
    least, segments = 2 * chunks * cdiv(one, CUS), 0
    for rounds in range(1, 5):
        for n in (CUS * rounds // both, CUS * rounds // one):
            n = min(n, chunks // 4)
            if n >= 2 and (t := 2 * cdiv(chunks, n) * (cdiv(both * n, CUS) + cdiv(one * n, CUS)) + n + 4) < least:
                least, segments = t, n
    segment = cdiv(chunks, segments) if segments else 0
    parts = sequences if not segment else slots // segment + sequences if packed else batch * cdiv(cdiv(time, CHUNK), segment)
    return slots, segment, parts, width, columns


def asked(batch, time, heads, key_dim, value_dim, packed, bwd, dtype):
    a = _delta.Delta(dtype=dtype, key_heads=1, heads=heads, key_dim=key_dim, value_dim=value_dim, batch=batch, time=time, sequences=packed or batch)
    a.cu_seqlens = 16 if packed else None  # (not read)
    return _delta._lib.linrec_delta_scratch_bytes(ctypes.byref(a), bwd)


CASES = [(1, 100001, 1, 64, 32, 3), (1, 8192, 4, 128, 128, 2), (1, 20011, 16, 128, 128, 37), (1, 4096, 1, 16, 16, 3), (1, 40000, 2, 200, 72, 5),
         (1, 8192, 16, 128, 128, 0), (3, 1700, 2, 100, 72, 0), (8, 4096, 16, 128, 128, 0), (1, 1, 1, 1, 1, 1), (1, 0, 2, 8, 8, 4)]


@pytest.mark.parametrize("case", CASES)
def test_the_library_asks_for_what_the_rule_says(case):
    batch, time, heads, *_ = case
    slots, segment, parts, width, columns = sizes(*case)
    for dtype in (0, 1, 2):
        for bwd in (0, 1):
            of_chunk = [16384, 16384, 768] + ([512, 16384, 4 * columns * width, 4 * columns * width, 256 * columns, 256 * columns, 768] if bwd else [])
            need = sum(cdiv(slots * heads * n, 256) * 256 for n in of_chunk)
            if segment:
                need += sum(cdiv(4 * parts * heads * n * width, 256) * 256 for n in (columns + width, columns))
            assert asked(*case, bwd, dtype) == need


def test_some_of_the_cases_are_cut():
    assert [bool(sizes(*c)[1]) for c in CASES] == [True, True, False, True, True, True, True, False, False, False]


def numbered(bounds, time, slots, segment, parts):
    """Checks what the kernels make of `bounds`, as they clamp them, and returns the numbers of chunks and of segments that they use."""
    chunks_used, parts_used = [], []
    for n in range(len(bounds) - 1):
        first, end = (min(max(b, 0), time) for b in bounds[n:n + 2])
        end = max(first, end)
        slot, chunks = first // CHUNK + n, cdiv(end - first, CHUNK)
        assert 0 <= slot and slot + chunks <= slots and first + (chunks - 1) * CHUNK < end or chunks == 0 and slot < slots
        chunks_used += range(slot, slot + chunks)
        if segment:
            at, count = slot // segment + n, cdiv(chunks, segment) if chunks > segment else 1
            assert 0 <= at and at + count <= parts
            parts_used += range(at, at + count)
    return chunks_used, parts_used


@pytest.mark.parametrize("case", [c for c in CASES if c[5]])
def test_every_chunk_and_segment_has_a_place(case):
    batch, time, heads, key_dim, value_dim, sequences = case
    slots, segment, parts, *_ = sizes(*case)
    rng = random.Random(time)
    for _ in range(300):
        ascending = [0] + sorted(rng.randint(0, time) for _ in range(sequences - 1)) + [time]
        for used in numbered(ascending, time, slots, segment, parts):
            assert len(set(used)) == len(used)  # no two sequences meet
        wrong = [rng.choice([rng.randint(0, time), rng.randint(-2 ** 31, 2 ** 31 - 1), 0, time]) for _ in range(sequences + 1)]
        numbered(wrong, time, slots, segment, parts)


def test_a_room_that_is_too_small_would_be_seen():
    slots, segment, parts, *_ = sizes(1, 8192, 4, 128, 128, 2)
    with pytest.raises(AssertionError):  # without a segment more for each sequence
        for n in range(0, 8193, 64):
            numbered([0, n, 8192], 8192, slots, segment, parts - 2)
