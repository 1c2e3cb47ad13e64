"""Edges of the 8-bit KV cache operators (GPU): masked keys whose scores scale to 0 or change sign.

Against the float64 restatements of test_kv8_gpu.py, whose tolerances count roundings.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

from pythonintern_b200 import _lib, kernels  # noqa: E402
from test_kv8_gpu import (DEV, _attend64, _close, _status_clean, _stored, _tables_for, gen, i32)  # noqa: E402,F401


def _check_rows(out, q, cache, tab, rows, scale, dtype):
    """out[r] against 64 bits for every (row, table row, keys seen)."""
    for r, s, upto in rows:
        want, size = _attend64(q[r], cache, 0, tab[s].tolist(), upto, scale)
        _close(out[r], want, size, dtype)


def _decode(q, nq, nkv, hd, cache, tab, ctx, scale):
    out = kernels.paged_attention_q8(q, nq, nkv, hd, *cache, 0, torch.from_numpy(tab).to(DEV), None, i32(ctx), False,
                                     scale)
    _lib.check_device_status(DEV, "decode")
    return out


def _prefill(q, nq, nkv, hd, cache, tab, lens, ctx0, scale):
    start = [0]
    for n in lens:
        start.append(start[-1] + n)
    out = kernels.prefill_attention_q8(q, nq, nkv, hd, *cache, 0, torch.from_numpy(tab).to(DEV), i32(start), len(lens),
                                       scale, seq_ctx0=i32(ctx0))
    _lib.check_device_status(DEV, "prefill")
    return out, [(start[s] + i, s, ctx0[s] + i + 1) for s, n in enumerate(lens) for i in range(n)]


SHAPES = [(8, 2, 128), (4, 2, 64), (3, 1, 32), (9, 1, 64)]
CTX = [1, 15, 16, 17, 31, 32, 40, 63]


def _masked_inputs(what, code, dtype, nq, nkv, hd, B, seen, seed):
    """A cache and queries whose scores in the last, partly seen block are scaled by 0, by next to 0 or by a
    negative number; the scale of the scores."""
    tab, NB = _tables_for([-(-c // 16) for c in seen], 2, seed)
    cache = _stored(code, NB, nkv, hd, seed=seed)
    q = torch.randn(B, nq * hd, generator=gen(seed + 1))
    scale = 1 / math.sqrt(hd)
    if what == "zero tile":      # a K tile of zeros; codes behind the context are whatever the block held before
        for s, c in enumerate(seen):
            b = int(tab[s, (c - 1) // 16])
            cache[2][0, b] = 0
            keep = (c - 1) % 16 + 1
            cache[0][0, b].view(torch.uint8)[:, :keep] = 0
    elif what == "zero head":
        q.view(B, nq, hd)[:, ::2] = 0
        cache[2] *= 2.0 ** -6    # tile maxima below 3.5
    elif what == "subnormal head":
        q.view(B, nq, hd)[:, ::2] *= 2.0 ** -128
        cache[2] *= 2.0 ** -6
    elif what == "scale 0":
        scale = 0.0
    else:
        scale = -scale
    return tab, cache, q.to(DEV, dtype), scale


WHAT = ["zero tile", "zero head", "subnormal head", "scale 0", "negative scale"]


@pytest.mark.parametrize("what", WHAT)
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_keys_of_a_decode_row_stay_masked(what, code, dtype):
    for nq, nkv, hd in SHAPES:
        tab, cache, q, scale = _masked_inputs(what, code, dtype, nq, nkv, hd, len(CTX), CTX, nq)
        out = _decode(q, nq, nkv, hd, cache, tab, CTX, scale)
        _check_rows(out, q, cache, tab, [(r, r, c) for r, c in enumerate(CTX)], scale, dtype)


@pytest.mark.parametrize("what", WHAT)
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_keys_of_a_prefill_row_stay_masked(what, code, dtype):
    lens, ctx0 = [1, 15, 16, 3, 5], [0, 0, 0, 28, 43]
    for nq, nkv, hd in SHAPES:
        seen = [c + n for c, n in zip(ctx0, lens)]
        tab, cache, q, scale = _masked_inputs(what, code, dtype, nq, nkv, hd, sum(lens), seen, nq)
        out, rows = _prefill(q, nq, nkv, hd, cache, tab, lens, ctx0, scale)
        _check_rows(out, q, cache, tab, rows, scale, dtype)


@pytest.mark.parametrize("what", WHAT)
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_masked_keys_of_many_prefill_rows_stay_masked(what, code):
    """Enough rows for the tcgen05 kernel (a scale of 0 or below stays with the other one)."""
    nq, nkv, hd, lens, ctx0 = 32, 16, 128, [200, 250], [33, 7]
    seen = [c + n for c, n in zip(ctx0, lens)]
    tab, cache, q, scale = _masked_inputs(what, code, torch.bfloat16, nq, nkv, hd, sum(lens), seen, 5)
    out, rows = _prefill(q, nq, nkv, hd, cache, tab, lens, ctx0, scale)
    _check_rows(out, q, cache, tab, rows[::23] + rows[190:202] + rows[-12:], scale, torch.bfloat16)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_a_scale_next_to_0_weighs_all_keys_alike(code):
    """scale * K scale rounds to 0: every visible key has the same score, the masked ones none."""
    nq, nkv, hd, scale = 32, 16, 128, 1e-44
    for lens, ctx0 in (([200, 250], [33, 7]), ([3, 2], [30, 7])):
        tab, NB = _tables_for([-(-(c + n) // 16) for c, n in zip(ctx0, lens)], 2, 1)
        cache = _stored(code, NB, nkv, hd, seed=2)
        q = torch.randn(sum(lens), nq * hd, generator=gen(3)).to(DEV, torch.bfloat16)
        out, rows = _prefill(q, nq, nkv, hd, cache, tab, lens, ctx0, scale)
        _check_rows(out, q, cache, tab, rows[::23] + rows[-5:], scale, torch.bfloat16)


# ------------------------------------------------------------------ value tiles of scale 0 under the loudest keys
def _loud_zero_values(code, nkv, hd, blocks, loud, gap, seed):
    """One sequence of `blocks` full blocks whose keys score -gap / 2 bits, but for block `loud`: +gap / 2, and a
    value tile of zeros.  Queries of all ones score so with scale 1."""
    tab, NB = _tables_for([blocks], 2, seed)
    cache = _stored(code, NB, nkv, hd, seed=seed)
    cache[0].zero_()
    one = 64 if code == "int8" else 0x38  # e4m3: 1.0
    cache[0].view(torch.uint8)[...] = (256 - one) if code == "int8" else one | 0x80
    cache[2].fill_(gap / 2 * math.log(2) / hd / (64 if code == "int8" else 1))
    b = int(tab[0, loud])
    cache[0].view(torch.uint8)[0, b] = one
    cache[1].view(torch.uint8)[0, b] = 0
    cache[3][0, b] = 0
    return tab, cache


def _close_to_next_to_nothing(got, want, size, cache, dtype):
    """As _close, for weights far below 1.  Scores of up to 2^7 bits err by 2^-14 of a weight.  The value reference
    is held within 2^100 of the score reference, where the loudest key weighs 2^8 or more: float16's half step of
    2^-25 leaves 2^-133 of a code, and a weight whose exponential is below 2^-126 counts as 0 (2^-134 of a value).
    The output's own half step below its normal numbers is 2^-134 (bf16) or 2^-150."""
    size, small = size
    out = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    prob = 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -22
    code = cache[1].double().abs().sum((2, 3, 4)).max().item()
    value = code * cache[3].double().max().item()
    assert torch.isfinite(got).all()
    limit = (out * want.abs() + (prob + 2.0 ** -14) * size + 2.0 ** -33 * small + 2.0 ** -133 * code
             + 2.0 ** -134 * value + 2.0 ** -134)
    err = (got.double().cpu() - want).abs()
    assert (err <= limit * 1.01).all(), float((err / limit).max())


@pytest.mark.parametrize("gap", [40, 110, 131, 150, 260])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_zero_values_under_the_loudest_keys(code, dtype, gap):
    nq, nkv, hd = 4, 2, 64
    for blocks, loud in ((2, 0), (2, 1), (10, 0), (10, 5), (10, 9), (300, 7)):
        tab, cache = _loud_zero_values(code, nkv, hd, blocks, loud, gap, blocks)
        ctx = 16 * blocks
        q = torch.ones(3, nq * hd, dtype=dtype, device=DEV)
        want, size = _attend64(q[0], cache, 0, tab[0].tolist(), ctx, 1.0)
        out = kernels.paged_attention_q8(q, nq, nkv, hd, *cache, 0, torch.from_numpy(tab).to(DEV), i32([0, 0, 0]),
                                         i32([ctx] * 3), False, 1.0)
        _lib.check_device_status(DEV, "decode")
        _close_to_next_to_nothing(out[1], want, size, cache, dtype)
        out, rows = _prefill(q, nq, nkv, hd, cache, tab, [3], [ctx - 3], 1.0)
        _close_to_next_to_nothing(out[2], want, size, cache, dtype)


@pytest.mark.parametrize("gap", [40, 110, 131, 150, 260])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_zero_values_under_the_loudest_keys_of_many_rows(code, gap):
    """Enough rows for the tcgen05 kernel; the loud block in the first tile, within it behind others, and later."""
    nq, nkv, hd, blocks = 32, 16, 128, 25
    for loud in (0, 2, 3, 9, 24):
        tab, cache = _loud_zero_values(code, nkv, hd, blocks, loud, gap, blocks)
        n = 16 * blocks
        q = torch.ones(n, nq * hd, dtype=torch.bfloat16, device=DEV)
        out, rows = _prefill(q, nq, nkv, hd, cache, tab, [n], [0], 1.0)
        for r in (0, 15, 16, 63, 64, 200, n - 1):
            want, size = _attend64(q[r], cache, 0, tab[0].tolist(), r + 1, 1.0)
            _close_to_next_to_nothing(out[r], want, size, cache, torch.bfloat16)


# ------------------------------------------------------------------ maps that hold more than the step's tokens
@pytest.mark.parametrize("T", [96, 30001])
@pytest.mark.parametrize("refused", [False, True])
def test_map_entries_of_no_token_are_written_by_none(refused, T):
    """Without maps given, entries behind the step's tokens, and all of a refused call, name no token: a write that
    runs on them before the status is read leaves the cache as it was."""
    nq, nkv, hd, bs = 4, 2, 64, 16
    tables = torch.full((3, 4), -1, dtype=torch.int32, device=DEV)
    lens, ring, state = i32([0, 0, 0]), i32(list(range(12))), i32([0, 12, 0, 0])
    # the memory that the next maps get holds those of an earlier step
    m = kernels.block_tables_extend(tables, lens, i32([40, 16, 40]), T, bs, ring, state)
    del m
    new = [40, 0, 100] if refused else [1, 0, 2]
    m = kernels.block_tables_extend(tables, lens, i32(new), T, bs, ring, state)
    n = 0 if refused else 3
    assert (m.positions[n:] == -1).all() and (m.slots[n:] == -1).all()
    assert (m.table_index[n:] == 0).all() and (m.ctx_lens[n:] == 0).all()
    if refused:
        assert (m.seq_start == 0).all() and (m.last_rows == -1).all()
    else:
        assert m.positions[:3].tolist() == [40, 40, 41] and m.seq_start.tolist() == [0, 1, 1, 3]
    qkv = torch.randn(T, (nq + 2 * nkv) * hd, device=DEV).to(torch.bfloat16)
    cos = sin = torch.ones(64, hd, device=DEV)
    q = torch.empty(T, nq * hd, dtype=torch.bfloat16, device=DEV)
    cache = _stored("int8", 12, nkv, hd)
    before = [t.clone() for t in cache]
    kernels.qk_norm_rope_kv_write_q8(qkv, nq, nkv, hd, None, None, 1e-5, m.positions, None, m.table_index, tables, cos,
                                     sin, q, *cache, 0)
    touched = torch.zeros(12, dtype=torch.bool, device=DEV)
    if not refused:
        touched[tables[0, 2]] = touched[tables[2, 2]] = True
    for t, b in zip(cache, before):
        assert torch.equal(t[0][~touched], b[0][~touched])
    with pytest.raises((IndexError, MemoryError)):
        _lib.check_device_status(DEV, "write")


# ------------------------------------------------------------------ ids outside the pool in tables and ring
@pytest.mark.parametrize("bad", [-1, 12, 1 << 30])
def test_block_ids_outside_the_pool_are_reported(bad):
    """truncate over a table with a hole, and extend from a ring with one: the call reports it."""
    tables, lens = i32([[4, bad, 2], [7, 8, -1]]), i32([40, 32])
    ring, state = i32([0] * 12), i32([0, 0, 0, 0])
    kernels.block_tables_truncate(tables, lens, i32([0, 32]), 16, ring, state)
    with pytest.raises(IndexError):
        _lib.check_device_status(DEV, "truncate")
    assert lens.tolist() == [0, 32] and tables.tolist() == [[-1] * 3, [7, 8, -1]]
    # the hole takes its place in the ring as -1 ...
    assert state[:2].tolist() == [0, 3] and ring[:3].tolist() == [4, -1, 2]
    # ... and the sequence that draws it holds no block there
    m = kernels.block_tables_extend(tables, lens, i32([33, 0]), 33, 16, ring, state)
    with pytest.raises(IndexError):
        _lib.check_device_status(DEV, "extend")
    assert tables[0].tolist() == [4, -1, 2] and (m.slots[16:32] == -1).all() and m.slots[32] == 32
    ring2 = i32([bad] * 12)
    tables = i32([[-1, -1]])
    m = kernels.block_tables_extend(tables, i32([0]), i32([17]), 17, 16, ring2, i32([3, 12, 0, 0]))
    with pytest.raises(IndexError):
        _lib.check_device_status(DEV, "extend")
    assert (tables == -1).all() and (m.slots == -1).all()


# ------------------------------------------------------------------ arguments that the wrappers refuse or take
def _write_args(n=3, nq=4, nkv=2, hd=64, positions=32):
    qkv = torch.randn(n, (nq + 2 * nkv) * hd, generator=gen(1)).to(DEV, torch.bfloat16)
    pos = torch.arange(n, dtype=torch.int64, device=DEV)
    angle = torch.arange(positions)[:, None] / 10000.0 ** (torch.arange(hd // 2) * 2 / hd)
    cos, sin = (torch.cat([f, f], 1).to(DEV) for f in (angle.cos(), angle.sin()))
    return dict(qkv=qkv, nq=nq, nkv=nkv, hd=hd, pos=pos, store=None, row=i32([0] * n), tab=i32([[1, 2]]), cos=cos, sin=sin)


def _run_write(a, q8, cache=None):
    """One write into a fresh cache (or the given one): q, and what it wrote."""
    q = torch.zeros(a["qkv"].shape[0], a["nq"] * a["hd"], dtype=a["qkv"].dtype, device=DEV)
    head = (a["qkv"], a["nq"], a["nkv"], a["hd"], None, None, 1e-5, a["pos"], a["store"], a["row"], a["tab"], a["cos"],
            a["sin"], q)
    if q8:
        cache = _stored("int8", 4, a["nkv"], a["hd"]) if cache is None else cache
        kernels.qk_norm_rope_kv_write_q8(*head, *cache, 0)
    else:
        cache = list(torch.zeros(2, 1, 4, 16, a["nkv"], a["hd"], dtype=a["qkv"].dtype, device=DEV).unbind(0))
        kernels.qk_norm_rope_kv_write(*head, *cache, 0)
    return [q] + cache


@pytest.mark.parametrize("q8", [False, True])
def test_rotation_tables_of_another_shape_are_refused(q8):
    """The kernel reads cos and sin as rows of head_dim for as many positions as cos has rows."""
    a = _write_args()
    _run_write(a, q8)
    c, s = a["cos"], a["sin"]
    for bad in (dict(cos=c[0], sin=s[0]), dict(cos=c.view(-1), sin=s.view(-1)), dict(cos=c[:, :32].contiguous()),
                dict(cos=c[:, :32].contiguous(), sin=s[:, :32].contiguous()), dict(sin=s[:16]), dict(cos=c[None]),
                dict(sin=s.view(-1)), dict(cos=torch.cat([c, c], 1), sin=torch.cat([s, s], 1)), dict(sin=s.double())):
        with pytest.raises(_lib.B2Error):
            _run_write({**a, **bad}, q8)
    _lib.check_device_status(DEV, "refusals")


@pytest.mark.parametrize("q8", [False, True])
def test_a_single_row_may_have_any_stride(q8):
    a = _write_args(n=1)
    want = _run_write(a, q8)
    width = a["qkv"].shape[1]
    odd = torch.zeros(3, width + 3, dtype=torch.bfloat16, device=DEV)
    row = torch.as_strided(odd, (1, width), (width + 3, 1))
    wide = torch.as_strided(odd, (1, width + 3), (width + 3, 1))  # columns behind the heads, an odd number
    for qkv in (row, wide):
        qkv[:, :width] = a["qkv"]
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8))
                   for x, y in zip(_run_write({**a, "qkv": qkv}, q8), want))
    _lib.check_device_status(DEV, "write")


def test_a_single_query_row_may_have_any_stride():
    nq, nkv, hd, ctx = 4, 2, 64, 40
    tab, NB = _tables_for([3], 1, 1)
    cache, t = _stored("int8", NB, nkv, hd), torch.from_numpy(tab).to(DEV)
    q = torch.randn(1, nq * hd, generator=gen(2)).to(DEV, torch.bfloat16)
    want = _decode(q, nq, nkv, hd, cache, tab, [ctx], 0.1)
    pre, _ = _prefill(q, nq, nkv, hd, cache, tab, [1], [ctx - 1], 0.1)
    wide = torch.zeros(1, nq * hd + 5, dtype=torch.bfloat16, device=DEV)
    wide[:, :nq * hd] = q
    out = torch.full((3, nq * hd + 5), 7.0, dtype=torch.bfloat16, device=DEV)
    kernels.paged_attention_q8(wide, nq, nkv, hd, *cache, 0, t, None, i32([ctx]), False, 0.1, out=out)
    assert torch.equal(out[:1, :nq * hd], want) and (out[1:] == 7).all() and (out[0, nq * hd:] == 7).all()
    out.fill_(7)
    kernels.prefill_attention_q8(wide, nq, nkv, hd, *cache, 0, t, i32([0, 1]), 1, 0.1, seq_ctx0=i32([ctx - 1]), out=out)
    assert torch.equal(out[:1, :nq * hd], pre) and (out[1:] == 7).all() and (out[0, nq * hd:] == 7).all()
    _lib.check_device_status(DEV, "attention")


@pytest.mark.parametrize("nq,nkv,T", [(32, 16, 450), (4, 2, 20)])
def test_a_seq_start_that_leaves_the_rows_or_goes_back_is_reported(nq, nkv, T):
    """In the tcgen05 kernel (450 rows) and the other one; where it names more tokens than there are rows, nothing is
    computed."""
    hd = 128
    tab, NB = _tables_for([T // 16 + 2] * 3, 1, 1)
    cache, t = _stored("int8", NB, nkv, hd), torch.from_numpy(tab).to(DEV)
    q = torch.randn(T, nq * hd, generator=gen(2)).to(DEV, torch.bfloat16)
    half = T // 2
    for start, nothing in (([0, 1 << 30, 1 << 30, 1 << 30], True), ([0, 2 ** 31 - 1, 0, T], False),
                           ([0, T, half, T], False), ([0, half, half - 1, half], False), ([-5, half, half, T], False),
                           ([0, half, T, T + 1], False)):
        out = torch.full((T, nq * hd), 7.0, dtype=torch.bfloat16, device=DEV)
        kernels.prefill_attention_q8(q, nq, nkv, hd, *cache, 0, t, i32(start), 3, 0.1, out=out)
        with pytest.raises(IndexError):
            _lib.check_device_status(DEV, "prefill")
        assert torch.isfinite(out).all() and (not nothing or (out == 7).all())


# ------------------------------------------------------------------ positions in the cache and in the rotation tables
def _tokens(lens, ctx0, positions, nq=4, nkv=2, hd=64):
    a = _write_args(sum(lens), nq, nkv, hd, positions)
    a["pos"] = torch.cat([torch.arange(c, c + n) for c, n in zip(ctx0, lens)]).to(DEV)
    a["row"] = torch.arange(len(lens)).repeat_interleave(torch.tensor(lens)).to(DEV, torch.int32)
    width = max(-(-(c + n) // 16) for c, n in zip(ctx0, lens))
    a["tab"] = torch.randperm(width * len(lens), generator=gen(4)).to(DEV, torch.int32).view(len(lens), width)
    return a


def _write_into(a, q8, rows=slice(None)):
    NB = a["tab"].numel()
    if q8:
        cache = _stored("int8", NB, a["nkv"], a["hd"], seed=3)
    else:
        cache = list(torch.full((2, 1, NB, 16, a["nkv"], a["hd"]), 3.0, dtype=torch.bfloat16, device=DEV).unbind(0))
    q = torch.full((a["qkv"].shape[0], a["nq"] * a["hd"]), 9.0, dtype=torch.bfloat16, device=DEV)
    some = {k: a[k][rows].contiguous() for k in ("qkv", "pos", "row")}
    store = None if a["store"] is None else a["store"][rows].contiguous()
    part = q[rows].contiguous()
    fn = kernels.qk_norm_rope_kv_write_q8 if q8 else kernels.qk_norm_rope_kv_write
    fn(some["qkv"], a["nq"], a["nkv"], a["hd"], None, None, 1e-5, some["pos"], store, some["row"], a["tab"], a["cos"],
       a["sin"], part, *cache, 0)
    q[rows] = part
    return [q] + cache


@pytest.mark.parametrize("q8", [False, True])
def test_tokens_are_rotated_by_one_position_and_stored_at_another(q8):
    """store_pos gives the slots, rope_pos the angles: the same, bit for bit, as tables whose rows are put in the
    order of the slots."""
    a = _tokens([20, 15, 33, 1], [0, 25, 64, 48], 100)
    order = torch.randperm(100, generator=gen(7)).to(DEV)
    split = {**a, "pos": order[a["pos"]], "store": a["pos"]}
    assert (split["pos"] != split["store"]).any()
    joint = {**a, "cos": a["cos"][order].contiguous(), "sin": a["sin"][order].contiguous()}
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8))
               for x, y in zip(_write_into(split, q8), _write_into(joint, q8)))
    _lib.check_device_status(DEV, "write")


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("positions", [20, 32, 33, 40])
def test_tokens_past_the_rotation_tables_leave_no_trace(q8, positions):
    """Their q rows, slots and blocks stay as they were, and all other tokens are written as without them."""
    a = _tokens([5, 20, 3], [0, 25, 7], positions)
    good = a["pos"] < positions
    want = _write_into(a, q8, good)
    _lib.check_device_status(DEV, "write")
    got = _write_into(a, q8)
    with pytest.raises(IndexError):
        _lib.check_device_status(DEV, "write")
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(got, want))


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("what", ["row", "block", "position"])
def test_tokens_without_a_slot_leave_the_others_right(q8, what):
    """A sequence whose table row or block is not there, and tokens of no position behind the last one."""
    a = _tokens([5, 20, 3, 4], [0, 12, 7, 16], 64)
    good = torch.ones(32, dtype=torch.bool, device=DEV)
    if what == "row":
        a["row"][-4:] = 4
        good[-4:] = False
    elif what == "block":
        a["tab"][1, 1] = 1 << 20  # positions 16..31 of the second sequence, 12..31
        good[9:25] = False
    else:
        a["pos"][-4:] = -1
        good[-4:] = False
    want = _write_into(a, q8, good)
    want_q = _write_into({**a, "tab": torch.arange(8, device=DEV, dtype=torch.int32).view(4, 2),
                          "row": a["row"].clamp(max=3)}, q8)[0]
    if what == "position":
        with pytest.raises(IndexError):
            _lib.check_device_status(DEV, "write")
    _lib.check_device_status(DEV, "write")
    got = _write_into(a, q8)
    with pytest.raises(IndexError):
        _lib.check_device_status(DEV, "write")
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(got[1:], want[1:]))
    assert torch.equal(got[0], want_q)  # a token without a slot still has its q, one without a position does not
