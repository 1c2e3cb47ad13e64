"""Host restatement of the 8-bit tcgen05 prefill kernel's converter stage (CPU).

`pythonintern_b200/csrc/prefill_q8_tc.cu` has converter warps in the producer's place for K and
V: they read codes into registers, widen them into a three-stage operand ring, and the MMA
warp releases operand stages by commits.  Checked here: the protocol finishes under
random completion orders and no stage is rewritten before its readers are done; the converter threads cover every piece of a tile once, store it where the swizzled
operand has it, and without bank conflicts; the bit tricks that widen a code are exact.
"""

import random

import numpy as np
import pytest
from test_prefill_tc_schedule import Bar, items

NG, ST, GW, CW = 2, 3, 4, 2


def simulate(work, seed):
    rnd = random.Random(seed)
    q_full = [[Bar(1), Bar(1)] for _ in range(NG)]
    q_empty = [[Bar(GW), Bar(GW)] for _ in range(NG)]  # handed back by the epilogue, which stages rows there
    kv_full, kv_empty = [Bar(CW) for _ in range(ST)], [Bar(1) for _ in range(ST)]
    s_full = [[Bar(1), Bar(1)] for _ in range(NG)]
    p_full = [[Bar(GW), Bar(GW)] for _ in range(NG)]
    pv_done = [[Bar(1), Bar(1)] for _ in range(NG)]
    o_empty = [Bar(GW) for _ in range(NG)]
    pending, commits = [], []                    # copies in any order; commits in issue order
    kv_tile = [[None] * CW for _ in range(ST)]   # the tile whose operands a stage holds, per converter warp
    q_given = [[0] * GW for _ in range(NG)]      # Q tiles handed back, per softmax warp
    kv_done = set()                              # tiles whose PV MMAs have completed

    def producer():
        iq = [0, 0]
        for tiles in work:
            for g in range(NG):
                if tiles[g][1] == 0:
                    continue
                while not q_empty[g][iq[g] & 1].ready(((iq[g] >> 1) & 1) ^ 1):
                    yield
                assert min(q_given[g]) >= iq[g] - 1, "Q overwritten before the epilogue was done with it"
                pending.append(q_full[g][iq[g] & 1])
                iq[g] += 1

    def converter(w):
        J = 0
        for tiles in work:
            for _ in range(tiles[0][2]):
                st = J % ST
                while not kv_empty[st].ready(((J // ST) & 1) ^ 1):
                    yield
                assert J < ST or J - ST in kv_done, "operands overwritten before the MMAs read them"
                kv_tile[st][w] = J
                kv_full[st].arrive()
                J += 1
                if rnd.random() < 0.3:
                    yield

    def mma():
        iq, js, jp, io, J = [0, 0], [0, 0], [0, 0], [0, 0], 0

        def issue_pv(g, first):
            while not p_full[g][jp[g] & 1].ready((jp[g] >> 1) & 1):
                yield
            if first:
                while not o_empty[g].ready((io[g] & 1) ^ 1):
                    yield
                io[g] += 1
            commits.append((pv_done[g][jp[g] & 1], None))
            jp[g] += 1

        for tiles in work:
            n_kv = [t[2] for t in tiles]
            qb = [0, 0]
            for g in range(NG):
                if tiles[g][1] == 0:
                    continue
                qb[g] = iq[g] & 1
                while not q_full[g][qb[g]].ready((iq[g] >> 1) & 1):
                    yield
                iq[g] += 1
            for j in range(n_kv[0]):
                st = J % ST
                while not kv_full[st].ready((J // ST) & 1):
                    yield
                assert kv_tile[st] == [J] * CW
                for g in range(NG):
                    if j < n_kv[g]:
                        commits.append((s_full[g][js[g] & 1], None))
                        js[g] += 1
                if j >= 1:
                    for g in range(NG):
                        if j - 1 < n_kv[g]:
                            yield from issue_pv(g, j == 1)
                    assert kv_tile[(J - 1) % ST] == [J - 1] * CW
                    commits.append((kv_empty[(J - 1) % ST], J - 1))
                J += 1
            for g in range(NG):
                if n_kv[g] == n_kv[0] and n_kv[0] > 0:
                    yield from issue_pv(g, n_kv[0] == 1)
            commits.append((kv_empty[(J - 1) % ST], J - 1))

    def softmax(grp, wid):
        js = 0
        for tiles in work:
            if tiles[grp][1] == 0:
                continue
            for _ in range(tiles[grp][2]):
                while not s_full[grp][js & 1].ready((js >> 1) & 1):
                    yield
                p_full[grp][js & 1].arrive()
                js += 1
            while not pv_done[grp][(js - 1) & 1].ready(((js - 1) >> 1) & 1):
                yield
            o_empty[grp].arrive()
            if rnd.random() < 0.5:
                yield
            q_given[grp][wid] += 1
            q_empty[grp][(q_given[grp][wid] - 1) & 1].arrive()

    roles = [producer(), mma()] + [converter(w) for w in range(CW)] + [softmax(g, w) for g in range(NG) for w in range(GW)]
    alive = list(range(len(roles)))
    for _ in range(3_000_000):
        if not alive:
            return True
        if pending and rnd.random() < 0.3:
            pending.pop(rnd.randrange(len(pending))).arrive()
        if commits and rnd.random() < 0.3:
            bar, tile = commits.pop(0)
            if tile is not None:
                kv_done.add(tile)
            bar.arrive()
        r = rnd.choice(alive)
        try:
            next(roles[r])
        except StopIteration:
            alive.remove(r)
    return False


@pytest.mark.parametrize("qt", [16, 18, 32, 128])
@pytest.mark.parametrize("lens,ctx0", [([1], [0]), ([5, 130, 77], [0, 17, 0]), ([300, 1, 64, 65], [200, 0, 0, 9])])
def test_protocol_finishes_without_early_reuse(qt, lens, ctx0):
    work = [tiles for _, _, tiles in items(lens, ctx0, qt, 1)]
    for seed in range(3):
        assert simulate(work, seed)


def _piece(c, i):
    """(key, half, 16-dim chunk of the half) of piece i of converter thread c."""
    return (c >> 4) * 2 + ((c >> 2) & 1) + 8 * i, (c >> 3) & 1, c & 3


def test_converter_threads_cover_a_tile_once_and_without_bank_conflicts():
    seen = set()
    for i in range(8):
        for c0 in range(0, 32 * CW, 8):
            for second in range(2):
                banks = set()
                for c in range(c0, c0 + 8):
                    key, half, ch = _piece(c, i)
                    assert 0 <= key < 64 and key // 16 == i // 2
                    x = ((2 * ch + second) ^ (key & 7)) * 16
                    at = half * 8192 + key * 128 + x
                    # the 128-byte swizzle: 16-byte chunk index xor the row's low three bits
                    assert x // 16 ^ (at >> 7 & 7) == 2 * ch + second
                    banks.add(at // 16 % 8)
                    seen.add((key, half, 2 * ch + second))
                assert len(banks) == 8
    assert seen == {(k, h, x) for k in range(64) for h in range(2) for x in range(8)}


def _bf16(bits):
    return (np.asarray(bits, dtype=np.uint32) << 16).view(np.float32)


def test_widening_int8_is_exact():
    code = np.arange(-128, 128)
    byte = code.astype(np.int8).view(np.uint8).astype(np.uint32)
    low = _bf16(0x4300 | (byte & 0x7f))
    sign = _bf16(0x4300 | (byte & 0x80))
    assert np.array_equal(low - sign, code.astype(np.float32))
    assert np.array_equal(_bf16((code.astype(np.float32)).view(np.uint32) >> 16), code)  # representable in bf16
    half = (0x6400 | (byte ^ 0x80)).astype(np.uint16).view(np.float16).astype(np.float32) - 1152
    assert np.array_equal(half, code.astype(np.float32))
