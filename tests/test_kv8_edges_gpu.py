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
