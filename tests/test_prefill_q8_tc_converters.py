"""The converter stage of `pythonintern_b200/csrc/prefill_q8_tc.cu` as the kernel has it (CPU).

Warps, stages and tile sizes are read from the sources, so that this restatement follows them: the barrier protocol
with that many converter warps, and the pieces of a K/V tile that their threads widen and store.
"""

import os
import re

import pytest
import test_prefill_q8_tc_schedule as schedule
from pythonintern_b200 import build
from test_prefill_tc_schedule import items


def _const(name, file="prefill_q8_tc.cu"):
    text = open(os.path.join(build.CSRC, file)).read()
    return int(re.search(rf"constexpr \w+ {name} = (\d+);", text).group(1))


WARPS, KT, HD = _const("kConvertWarps"), _const("KT", "prefill_tc.cuh"), _const("HD", "prefill_tc.cuh")
PIECES = KT * HD // 16 // (32 * WARPS)
KEYS = KT // PIECES


def test_the_sources_constants():
    assert (WARPS, _const("ST"), KT, HD, PIECES, KEYS) == (4, schedule.ST, 64, 128, 4, 16)
    assert (_const("NG", "prefill_tc.cuh"), _const("kGroupWarps", "prefill_tc.cuh")) == (schedule.NG, schedule.GW)
    assert 16 % KEYS == 0  # a thread's pieces of one block follow each other


@pytest.mark.parametrize("qt", [16, 18, 32, 128])
@pytest.mark.parametrize("lens,ctx0", [([1], [0]), ([5, 130, 77], [0, 17, 0]), ([300, 1, 64, 65], [200, 0, 0, 9])])
def test_protocol_finishes_with_this_many_converter_warps(monkeypatch, qt, lens, ctx0):
    monkeypatch.setattr(schedule, "CW", WARPS)
    work = [tiles for _, _, tiles in items(lens, ctx0, qt, 1)]
    for seed in range(3):
        assert schedule.simulate(work, seed)


def _thread(c):
    """(half, first key, 16-dim chunk of the half) of converter thread c."""
    return (c >> 3) & 1, (c >> 4) * 2 + ((c >> 2) & 1), c & 3


def test_threads_read_and_store_every_piece_of_a_tile_once():
    read, stored = set(), set()
    for c in range(32 * WARPS):
        half, key0, ch = _thread(c)
        assert 0 <= key0 < KEYS
        for u in range(KT // 16):
            for i in range(16 // KEYS):
                # code[u * (16 / KEYS) + i]: block u, its key key0 + KEYS i
                piece, key = u * (16 // KEYS) + i, key0 + KEYS * i
                assert key < 16 and 16 * u + key == key0 + KEYS * piece
                read.add((u, key, half * 64 + ch * 16))
        for i in range(PIECES):
            for second in range(2):
                x = ((2 * ch + second) ^ (key0 & 7)) * 16
                at = half * KT * 128 + key0 * 128 + i * KEYS * 128 + x
                key = key0 + KEYS * i
                assert at // 128 % KT == key
                # the 128-byte swizzle: 16-byte chunk index xor the row's low three bits
                assert x // 16 ^ (at >> 7 & 7) == 2 * ch + second
                stored.add((key, half, 2 * ch + second))
    assert len(read) == KT * HD // 16 and len(stored) == KT * HD // 8
    assert read == {(u, k, d) for u in range(KT // 16) for k in range(16) for d in range(0, HD, 16)}


def test_no_store_phase_meets_a_bank_twice():
    for i in range(PIECES):
        for c0 in range(0, 32 * WARPS, 8):  # the eight threads of a 16-byte store phase
            for second in range(2):
                banks = set()
                for c in range(c0, c0 + 8):
                    half, key0, ch = _thread(c)
                    banks.add((half * KT * 128 + (key0 + KEYS * i) * 128 + ((2 * ch + second) ^ (key0 & 7)) * 16) // 16 % 8)
                assert len(banks) == 8
