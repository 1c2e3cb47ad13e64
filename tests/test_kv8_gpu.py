"""The 8-bit paged KV cache and the bookkeeping around it (GPU): block tables built on the
device, q/k norms + rotation + cache write, tile read-back and attention over the codes.

Checked against plain float64 restatements on the CPU.  Tolerances count roundings: half a
step is 2^-8 relative in bf16, 2^-11 in float16, 2^-24 in float32, 2^-4 in e4m3, and half a
scale step absolute in int8.
"""

import math
import random

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

from pythonintern_b200 import _lib, kernels  # noqa: E402
from pythonintern_b200.model.attention import RotaryEmbedding  # noqa: E402

DEV = torch.device("cuda", 0)
CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.fixture(autouse=True)
def _status_clean():
    _lib.check_device_status(DEV, "before test")
    yield
    torch.cuda.synchronize()


# ------------------------------------------------------------------ block tables
class HostTables:
    """The host bookkeeping: FIFO free list, tables, lengths."""

    def __init__(self, n, width, ring, head, count, bs):
        self.bs, self.n, self.width, self.pool = bs, n, width, len(ring)
        self.free = [ring[(head + i) % len(ring)] for i in range(count)]
        self.tables = [[] for _ in range(n)]
        self.lens = [0] * n

    def extend(self, new):
        pos, row, slots, start, last = [], [], [], [0], []
        for s, m in enumerate(new):
            while len(self.tables[s]) < -(-(self.lens[s] + m) // self.bs):
                self.tables[s].append(self.free.pop(0))
            for i in range(m):
                p = self.lens[s] + i
                pos.append(p)
                row.append(s)
                slots.append(self.tables[s][p // self.bs] * self.bs + p % self.bs)
            self.lens[s] += m
            start.append(start[-1] + m)
            last.append(start[-1] - 1 if m else -1)
        return start, pos, row, slots, last

    def truncate(self, keep):
        for s, k in enumerate(keep):
            k = min(k, self.lens[s])
            cut = -(-k // self.bs)
            self.free.extend(self.tables[s][cut:])
            del self.tables[s][cut:]
            self.lens[s] = k


def _device_tables(n, width, pool, bs, head, seed):
    ids = torch.randperm(pool, generator=gen(seed)).tolist()
    ring = i32(ids)
    return (torch.full((n, width), -1, dtype=torch.int32, device=DEV), i32([0] * n), ring, i32([head, pool, 0, 0]),
            HostTables(n, width, ids, head, pool, bs))


@pytest.mark.parametrize("n,width,bs,most,steps", [(1, 4, 16, 5, 12), (7, 9, 16, 40, 10), (130, 12, 16, 33, 6),
                                                   (300, 5, 1, 2, 5), (33, 20, 7, 50, 6), (2500, 3, 16, 9, 3)])
def test_block_tables_follow_the_host_bookkeeping(n, width, bs, most, steps):
    pool = n * width
    rng = random.Random(n)
    tables, lens, ring, state, host = _device_tables(n, width, pool, bs, pool - 1, n)
    for _ in range(steps):
        new = [min(rng.choice([0, 1, rng.randint(0, most)]), width * bs - host.lens[s]) for s in range(n)]
        total = sum(new)
        cap = total + 3
        out = kernels.SlotMap(*[torch.full((k,), -7, dtype=dt, device=DEV) for k, dt in (
            (n + 1, torch.int32), (cap, torch.int64), (cap, torch.int32), (cap, torch.int64), (cap, torch.int32),
            (n, torch.int64))])
        m = kernels.block_tables_extend(tables, lens, i32(new), cap, bs, ring, state, out=out)
        start, pos, row, slots, last = host.extend(new)
        tail = [-7] * 3
        assert m.seq_start.tolist() == start and m.positions.tolist() == pos + tail
        assert m.table_index.tolist() == row + tail and m.slots.tolist() == slots + tail
        assert m.ctx_lens.tolist() == [p + 1 for p in pos] + tail and m.last_rows.tolist() == last
        # the maps alone, of the same tokens: lens as they were before, nothing taken
        before = i32([a - b for a, b in zip(host.lens, new)])
        again = kernels.block_tables_extend(tables, before, i32(new), total, bs, num_blocks=pool)
        assert again.slots.tolist() == slots and again.positions.tolist() == pos
        assert before.tolist() == [a - b for a, b in zip(host.lens, new)]
        keep = [rng.choice([0, host.lens[s], rng.randint(0, host.lens[s] + 1)]) for s in range(n)]
        kernels.block_tables_truncate(tables, lens, i32(keep), bs, ring, state)
        host.truncate(keep)
        assert lens.tolist() == host.lens
        assert tables.tolist() == [t + [-1] * (width - len(t)) for t in host.tables]
        head, count, zero, _ = state.tolist()
        assert count == len(host.free) and zero == 0
        r = ring.tolist()
        assert [r[(head + i) % pool] for i in range(count)] == host.free
    _lib.check_device_status(DEV, "block tables")


def test_block_tables_long_sequence_and_graph_replay():
    tables, lens, ring, state, host = _device_tables(3, 400, 1000, 16, 990, 5)
    new, keep = i32([5000, 0, 6001]), i32([0, 0, 17])
    out = kernels.block_tables_extend(tables, lens, new, 11001, 16, ring, state)
    kernels.block_tables_truncate(tables, lens, keep, 16, ring, state)
    host.extend([5000, 0, 6001])
    host.truncate([0, 0, 17])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kernels.block_tables_extend(tables, lens, new, 11001, 16, ring, state, out=out)
        kernels.block_tables_truncate(tables, lens, keep, 16, ring, state)
    for vals in ([10, 3, 0], [0, 31, 5000]):
        new.copy_(i32(vals))
        g.replay()
        start, pos, row, slots, last = host.extend(vals)
        host.truncate([0, 0, 17])
        assert out.slots[:sum(vals)].tolist() == slots and out.last_rows.tolist() == last
        assert lens.tolist() == host.lens


@pytest.mark.parametrize("what", ["blocks", "width", "tokens", "negative", "state"])
def test_block_tables_refuse_whole(what):
    """A step that cannot be served changes nothing, maps included, and reports why."""
    tables, lens, ring, state, _ = _device_tables(4, 4, 12, 16, 3, 1)
    kernels.block_tables_extend(tables, lens, i32([20, 1, 0, 16]), 37, 16, ring, state)
    new, cap = [1, 1, 1, 1], 200
    if what == "blocks":
        new = [40, 40, 50, 30]
    elif what == "width":
        new[1] = 64
    elif what == "tokens":
        cap = 3
    elif what == "negative":
        new[2] = -1
    else:
        state[1] = 13
    before = [t.clone() for t in (tables, lens, ring, state)]
    out = kernels.block_tables_extend(tables, lens, i32(new), cap, 16, ring, state)
    out.slots.fill_(5)
    out = kernels.block_tables_extend(tables, lens, i32(new), cap, 16, ring, state, out=out)
    with pytest.raises(MemoryError if what == "blocks" else IndexError):
        _lib.check_device_status(DEV, "extend")
    assert (out.slots == 5).all()
    if what in ("negative", "state"):
        kernels.block_tables_truncate(tables, lens, i32([0, 0, -1 if what == "negative" else 0, 0]), 16, ring, state)
        with pytest.raises(IndexError):
            _lib.check_device_status(DEV, "truncate")
    assert all(torch.equal(a, b) for a, b in zip(before, (tables, lens, ring, state)))


def test_block_tables_maps_report_a_missing_block():
    tables = i32([[4, -1], [9, 1]])
    m = kernels.block_tables_extend(tables, i32([15, 0]), i32([2, 18]), 20, 16, num_blocks=9)
    with pytest.raises(IndexError):
        _lib.check_device_status(DEV, "maps")
    assert m.slots.tolist() == [4 * 16 + 15, -1] + [-1] * 16 + [16, 17]


def test_block_tables_refusals():
    tables, lens, ring, state, _ = _device_tables(2, 4, 8, 16, 0, 1)
    new = i32([1, 1])
    ok = (tables, lens, new, 2, 16, ring, state)
    for at, bad in ((0, tables.cpu()), (0, tables.long()), (0, tables.t()), (1, lens[:1]), (2, new.long()),
                    (3, -1), (4, 0), (5, ring.long()), (6, state[:2]), (6, None)):
        args = list(ok)
        args[at] = bad
        with pytest.raises((_lib.B2Error, RuntimeError)):
            kernels.block_tables_extend(*args)
    with pytest.raises(_lib.B2Error):
        kernels.block_tables_extend(tables, lens, new, 2, 16)
    big = torch.zeros(16385, 1, dtype=torch.int32, device=DEV)
    with pytest.raises(_lib.B2Error, match="16384"):
        kernels.block_tables_extend(big, big.view(-1), big.view(-1), 2, 16, num_blocks=4)
    _lib.check_device_status(DEV, "refusals")


# ------------------------------------------------------------------ norms + rotation + write
def _step(lens, ctx0, nq, nkv, hd, dtype, seed, extra=0, spare=3):
    """Tokens of several sequences: qkv rows (strided by `extra`), positions, tables over a permuted pool."""
    need = [max(1, -(-(c + n) // 16)) for c, n in zip(ctx0, lens)]
    NB = sum(need) + spare
    perm = torch.randperm(NB, generator=gen(seed)).tolist()
    tab = np.full((len(lens), max(need)), -1, dtype=np.int32)
    k = 0
    for s, n in enumerate(need):
        tab[s, :n] = perm[k:k + n]
        k += n
    T = sum(lens)
    wide = torch.randn(T, (nq + 2 * nkv) * hd + extra, generator=gen(seed + 1)).mul_(2).to(DEV, dtype)
    pos = np.concatenate([np.arange(c, c + n) for c, n in zip(ctx0, lens)]) if T else np.zeros(0)
    row = np.repeat(np.arange(len(lens)), lens)
    return (wide[:, : (nq + 2 * nkv) * hd], torch.tensor(pos, dtype=torch.int64, device=DEV),
            torch.tensor(row, dtype=torch.int32, device=DEV), torch.from_numpy(tab).to(DEV), NB)


def _norm_rotate64(x, w, eps, cos, sin):
    x = x.double()
    if w is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    h = x.shape[-1] // 2
    c, s = cos.double()[:, None], sin.double()[:, None]
    return x * c + torch.cat([-x[..., h:], x[..., :h]], -1) * s


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,hd,extra", [(32, 8, 128, 0), (7, 1, 64, 8), (6, 3, 32, 40), (5, 5, 128, 16)])
def test_write_without_norms_equals_rope_kv_write(dtype, nq, nkv, hd, extra):
    qkv, pos, row, tab, NB = _step([1, 17, 5, 33], [0, 3, 16, 31], nq, nkv, hd, dtype, 3, extra)
    rope = RotaryEmbedding(hd, 128, 10000.0, DEV)
    outs = []
    for fn in ("plain", "norm"):
        q = torch.full((qkv.shape[0], nq * hd), 9.0, dtype=dtype, device=DEV)
        k, v = torch.zeros(2, 2, NB, 16, nkv, hd, dtype=dtype, device=DEV).unbind(0)
        if fn == "plain":
            kernels.rope_kv_write(qkv, nq, nkv, hd, pos, None, row, tab, rope.cos_cached, rope.sin_cached, q, k, v, 1)
        else:
            kernels.qk_norm_rope_kv_write(qkv, nq, nkv, hd, None, None, 1e-5, pos, None, row, tab, rope.cos_cached,
                                          rope.sin_cached, q, k, v, 1)
        outs.append((q, k, v))
    _lib.check_device_status(DEV, "write")
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("dtype,half", [(torch.bfloat16, 2.0 ** -8), (torch.float32, 2.0 ** -24)])
@pytest.mark.parametrize("nq,nkv,hd,extra", [(32, 8, 128, 0), (7, 1, 64, 8), (9, 3, 32, 40)])
def test_write_with_norms(dtype, half, nq, nkv, hd, extra):
    lens, ctx0 = [1, 20, 2], [40, 0, 15]
    qkv, pos, row, tab, NB = _step(lens, ctx0, nq, nkv, hd, dtype, 5, extra)
    T = qkv.shape[0]
    rope = RotaryEmbedding(hd, 128, 10000.0, DEV)
    wq, wk = (1 + 0.3 * torch.randn(2, hd, generator=gen(2))).to(DEV).unbind(0)
    q = torch.empty(T, nq * hd, dtype=dtype, device=DEV)
    k, v = torch.zeros(2, 1, NB, 16, nkv, hd, dtype=dtype, device=DEV).unbind(0)
    store = pos + 1 if lens[0] == 1 else pos
    kernels.qk_norm_rope_kv_write(qkv, nq, nkv, hd, wq, wk, 1e-5, pos, pos, row, tab, rope.cos_cached,
                                  rope.sin_cached, q, k, v, 0)
    _lib.check_device_status(DEV, "write")
    x = qkv.reshape(T, -1, hd)
    cos, sin = rope.cos_cached[pos], rope.sin_cached[pos]
    want_q = _norm_rotate64(x[:, :nq], wq, 1e-5, cos, sin)
    want_k = _norm_rotate64(x[:, nq:nq + nkv], wk, 1e-5, cos, sin)
    blk = tab[row.long(), pos // 16].long()
    # in float32: the norm (sum of hd squares, rsqrt, three products) and the rotation's two
    # products and sum err by less than 16 half steps of the head's largest magnitude
    for got, want in ((q.view(T, nq, hd), want_q), (k[0][blk, pos % 16], want_k)):
        size = want.abs().amax(-1, keepdim=True)
        assert ((got.double() - want).abs() <= half * want.abs() + 2 * 16 * 2.0 ** -24 * size).all()
    assert torch.equal(v[0][blk, pos % 16], x[:, nq + nkv:])
    untouched = torch.ones(NB, 16, dtype=torch.bool, device=DEV)
    untouched[blk, pos % 16] = False
    assert (k[0][untouched] == 0).all() and (v[0][untouched] == 0).all()
    assert store is not None


@pytest.mark.parametrize("q8", [False, True])
def test_write_skips_and_reports_bad_tokens(q8):
    nq, nkv, hd = 4, 2, 64
    qkv, pos, row, tab, NB = _step([3, 4, 2], [0, 14, 3], nq, nkv, hd, torch.bfloat16, 7)
    rope = RotaryEmbedding(hd, 32, 10000.0, DEV)
    cases = []
    for at, tensor, value in ((1, pos, 32), (4, pos, -1), (8, row, 3), (8, row, -1), (0, tab, NB)):
        p, r, t = pos.clone(), row.clone(), tab.clone()
        {id(pos): p, id(row): r, id(tab): t}[id(tensor)].view(-1)[at] = value
        cases.append((p, r, t))
    for p, r, t in cases:
        q = torch.full((9, nq * hd), 9.0, dtype=torch.bfloat16, device=DEV)
        if q8:
            k, v = torch.full((2, 1, NB, nkv, 16, hd), 3, dtype=torch.int8, device=DEV).unbind(0)
            ks, vs = torch.full((2, 1, NB, nkv), 1e-3, device=DEV).unbind(0)
            kernels.qk_norm_rope_kv_write_q8(qkv, nq, nkv, hd, None, None, 1e-5, p, None, r, t, rope.cos_cached,
                                             rope.sin_cached, q, k, v, ks, vs, 0)
        else:
            k, v = torch.full((2, 1, NB, 16, nkv, hd), 3, dtype=torch.bfloat16, device=DEV).unbind(0)
            kernels.qk_norm_rope_kv_write(qkv, nq, nkv, hd, None, None, 1e-5, p, None, r, t, rope.cos_cached,
                                          rope.sin_cached, q, k, v, 0)
        with pytest.raises(IndexError):
            _lib.check_device_status(DEV, "write")
        used = set(t.view(-1).tolist()) & set(tab.view(-1).tolist())
        for b in set(range(NB)) - used:
            assert (k[0, b].float() == 3).all() and (v[0, b].float() == 3).all()


# ------------------------------------------------------------------ 8-bit tiles
def _e4m3_step(x):
    """Spacing of e4m3 numbers around x (float64)."""
    return torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)


def _caches(code, NB, nkv, hd, layers=1, seed=0, fill=None):
    dt = CODES[code][0]
    if fill is None:
        raw = torch.randint(0, 255, (2, layers, NB, nkv, 16, hd), generator=gen(seed), dtype=torch.uint8)
        raw[(raw == 127) | (raw == 255)] = 5  # no e4m3 NaN
    else:
        raw = torch.full((2, layers, NB, nkv, 16, hd), fill, dtype=torch.uint8)
    k, v = raw.to(DEV).view(dt).unbind(0)
    ks, vs = (torch.rand(2, layers, NB, nkv, generator=gen(seed + 1)) * 0.02 + 1e-3).to(DEV).unbind(0)
    return k, v, ks, vs


def _write(qkv, nq, nkv, hd, w, pos, row, tab, rope, cache, layer=0):
    q = torch.empty(qkv.shape[0], nq * hd, dtype=qkv.dtype, device=DEV)
    kernels.qk_norm_rope_kv_write_q8(qkv, nq, nkv, hd, w, w, 1e-5, pos, None, row, tab, rope.cos_cached,
                                     rope.sin_cached, q, *cache, layer)
    return q


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,hd,norm,lens,ctx0", [
    (32, 8, 128, True, [1, 17, 5, 33], [0, 3, 16, 31]),
    (7, 1, 64, False, [1] * 9, [0, 1, 15, 16, 17, 31, 5, 8, 100]),
    (6, 3, 32, True, [64, 16, 15], [0, 16, 1]),
    (4, 4, 128, True, [700, 1, 1500, 31], [9, 0, 0, 2]),   # past the size where blocks look for runs in chunks
])
def test_write_q8_tiles(code, dtype, nq, nkv, hd, norm, lens, ctx0):
    qkv, pos, row, tab, NB = _step(lens, ctx0, nq, nkv, hd, dtype, 11, 16)
    T, top = qkv.shape[0], CODES[code][1]
    rope = RotaryEmbedding(hd, 1600, 10000.0, DEV)
    w = (1 + 0.3 * torch.randn(hd, generator=gen(2))).to(DEV) if norm else None
    cache = _caches(code, NB, nkv, hd, layers=2, seed=4)
    before = [t.clone() for t in cache]
    q = _write(qkv, nq, nkv, hd, w, pos, row, tab, rope, cache, 1)
    _lib.check_device_status(DEV, "write")
    # q equals the other form's, bit for bit
    q2 = torch.empty_like(q)
    kc, vc = torch.zeros(2, 1, NB, 16, nkv, hd, dtype=dtype, device=DEV).unbind(0)
    kernels.qk_norm_rope_kv_write(qkv, nq, nkv, hd, w, w, 1e-5, pos, None, row, tab, rope.cos_cached, rope.sin_cached,
                                  q2, kc, vc, 0)
    assert torch.equal(q, q2)
    for a, b in zip(cache, before):
        assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8))  # the other layer
    x = qkv.reshape(T, -1, hd)
    new = (_norm_rotate64(x[:, nq:nq + nkv], w, 1e-5, rope.cos_cached[pos], rope.sin_cached[pos]), x[:, nq + nkv:].double())
    tabl, posl, rowl = tab.tolist(), pos.tolist(), row.tolist()
    touched = {}
    for t in range(T):
        touched.setdefault(tabl[rowl[t]][posl[t] // 16], []).append(t)
    for c in range(2):
        codes, scales, was, was_s = cache[c][1], cache[2 + c][1], before[c][1], before[2 + c][1]
        for b, toks in touched.items():
            y = new[c][toks].transpose(0, 1)  # [nkv, run, hd]
            off = posl[toks[0]] % 16
            fresh = y.abs().amax((1, 2)) / top
            want = torch.maximum(fresh, was_s[b].double()) if off else fresh
            s = scales[b].double()
            assert ((s - want).abs() <= want * 2.0 ** -18).all()  # norm + rotation + division in float32
            got = codes[b].double() * s[:, None, None]
            run = got[:, off:off + len(toks)]
            step = s[:, None, None] * (torch.ones_like(y) if code == "int8" else _e4m3_step(y / s[:, None, None]))
            assert ((run - y).abs() <= step / 2 + y.abs() * 2.0 ** -18 + want[:, None, None] * top * 2.0 ** -20).all()
            if off:
                old = was[b, :, :off].double() * was_s[b].double()[:, None, None]
                hist = got[:, :off]
                grown = (s > was_s[b].double())[:, None, None]
                step = s[:, None, None] * (torch.ones_like(old) if code == "int8" else _e4m3_step(old / s[:, None, None]))
                assert ((hist - old).abs() <= torch.where(grown, step / 2 + old.abs() * 2.0 ** -20, 0.0)).all()
            rest = slice(off + len(toks), 16)
            assert torch.equal(codes[b, :, rest].view(torch.uint8), was[b, :, rest].view(torch.uint8))
        other = torch.tensor([b for b in range(NB) if b not in touched], device=DEV)
        assert torch.equal(codes[other].view(torch.uint8), was[other].view(torch.uint8))
        assert torch.equal(scales[other], was_s[other])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_write_q8_token_by_token_stays_within_a_step_of_the_whole(code):
    """Sixteen one-token steps of growing size: every growth rounds the history again, by half a
    step of the scale of that moment, so an entry is off by less than the sum of those."""
    nq, nkv, hd, top = 2, 2, 64, CODES[code][1]
    qkv, pos, row, tab, NB = _step([16], [0], nq, nkv, hd, torch.float32, 2)
    qkv *= (1.3 ** torch.arange(16, device=DEV))[:, None]
    rope = RotaryEmbedding(hd, 32, 10000.0, DEV)
    cache = _caches(code, NB, nkv, hd)
    b = int(tab[0, 0])
    sums = torch.zeros(nkv, dtype=torch.float64, device=DEV)
    for i in range(16):
        _write(qkv[i:i + 1], nq, nkv, hd, None, pos[i:i + 1], row[i:i + 1], tab, rope, cache)
        s = cache[3][0, b].double()
        sums += s / 2 * (1.0 if code == "int8" else 32.0)  # e4m3: the largest step is 32 scales
    v = cache[1][0, b].double() * s[:, None, None]
    want = qkv.reshape(16, -1, hd)[:, nq + nkv:].double().transpose(0, 1)
    assert ((v - want).abs() <= sums[:, None, None] * (1 + 2.0 ** -16)).all()
    assert ((s - want.abs().amax((1, 2)) / top).abs() <= s * 2.0 ** -20).all()
    # the same token again changes nothing (a captured step runs once eagerly first)
    before = [t.clone() for t in cache]
    _write(qkv[15:], nq, nkv, hd, None, pos[15:], row[15:], tab, rope, cache)
    assert all(torch.equal(a.view(torch.uint8), c.view(torch.uint8)) for a, c in zip(cache, before))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_write_q8_zeros_tiny_and_non_finite(code):
    nq, nkv, hd = 1, 1, 32
    rope = RotaryEmbedding(hd, 64, 10000.0, DEV)
    qkv, pos, row, tab, NB = _step([4, 4, 4, 4], [0, 0, 0, 4], nq, nkv, hd, torch.float32, 2)
    x = qkv.view(16, 3, hd)
    x[0:4, 2] = 0.0
    x[4:8, 2] = 1e-39          # below 2^-126 * 127: stored as zeros
    x[9, 2, 5] = float("inf")
    x[12:16, 2] = 0.0          # zeros behind a history keep the history
    cache = _caches(code, NB, nkv, hd, seed=3)
    old = cache[1][0].clone(), cache[3][0].clone()
    _write(qkv, nq, nkv, hd, None, pos, row, tab, rope, cache)
    _lib.check_device_status(DEV, "write")
    b = tab[:, 0].tolist()
    for s in (0, 1):
        assert cache[3][0, b[s], 0] == 0 and (cache[1][0, b[s], 0, :4].float() == 0).all()
    assert torch.isnan(cache[3][0, b[2], 0])
    assert cache[3][0, b[3], 0] == old[1][b[3], 0]
    assert torch.equal(cache[1][0, b[3], 0, :4].view(torch.uint8), old[0][b[3], 0, :4].view(torch.uint8))
    assert (cache[1][0, b[3], 0, 4:8].float() == 0).all()
    # a poisoned tile stays NaN when it goes on, and is clean when the block begins anew
    one = qkv[:1].clone()
    one.view(3, hd)[2] = 1.0
    _write(one, nq, nkv, hd, None, i64([4]), i32([2]), tab, rope, cache)
    assert torch.isnan(cache[3][0, b[2], 0])
    _write(one, nq, nkv, hd, None, i64([0]), i32([2]), tab, rope, cache)
    assert torch.isfinite(cache[3][0, b[2], 0])


def i64(v):
    return torch.tensor(v, dtype=torch.int64, device=DEV)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nkv,hd,n", [(8, 128, 5), (1, 32, 1), (3, 64, 40), (2, 64, 0)])
def test_read_q8(code, dtype, nkv, hd, n):
    NB = 23
    cache = _caches(code, NB, nkv, hd, layers=2, seed=n)
    ids = torch.randint(0, NB, (n,), generator=gen(n)).to(torch.int32)
    k, v = kernels.kv_read_q8(*cache, 1, ids.to(DEV), dtype)
    for got, c, s in ((k, cache[0], cache[2]), (v, cache[1], cache[3])):
        want = (c[1].float() * s[1][:, :, None, None]).transpose(1, 2)[ids.long().to(DEV)].to(dtype)
        assert torch.equal(got, want)
    _lib.check_device_status(DEV, "read")
    if n:
        ids[0] = NB
        k, v = kernels.kv_read_q8(*cache, 0, ids.to(DEV), dtype)
        assert (k[0] == 0).all() and (v[0] == 0).all()
        with pytest.raises(IndexError):
            _lib.check_device_status(DEV, "read")


# ------------------------------------------------------------------ attention
def _stored(code, NB, nkv, hd, layers=1, seed=0):
    x = torch.randn(2, layers, NB, nkv, 16, hd, generator=gen(seed))
    loud = torch.rand(2, layers, NB, nkv, 1, 1, generator=gen(seed + 1)) * 3 + 0.2
    s = x.abs().amax((4, 5), keepdim=True) / CODES[code][1]
    x = x / s
    x = x.round().to(torch.int8) if code == "int8" else x.clamp(-448, 448).to(torch.float8_e4m3fn)
    s = (s * loud)[..., 0, 0]
    return [t.to(DEV) for t in (x[0], x[1], s[0], s[1])]


def _attend64(q, cache, layer, table, upto, scale, npad=0):
    """One query token [nq, hd] over the first `upto` keys of `table`, in float64: the result, and what its
    errors are measured by: sum of p |v|, and max(p vs) * sum of |code| (see _close)."""
    nkv, hd = cache[0].shape[2], cache[0].shape[4]
    q = q.double().cpu().view(nkv, -1, hd)
    nb = -(-upto // 16)
    ids = [b for b in table[:nb]]
    x = []
    for c, s in ((cache[0], cache[2]), (cache[1], cache[3])):
        t = torch.stack([c[layer, max(b, 0)].cpu().to(torch.float64) * s[layer, max(b, 0)].cpu().double()[:, None, None]
                         for b in ids]) if ids else torch.zeros(0, nkv, 16, hd, dtype=torch.float64)
        x.append(t.transpose(0, 1).reshape(nkv, -1, hd)[:, :upto])
    ok = torch.tensor([b >= 0 for b in ids], dtype=torch.bool).repeat_interleave(16)[:upto]
    s = torch.einsum("grd,gkd->grk", q, x[0]) * scale
    s = torch.where(ok, s, torch.tensor(-math.inf, dtype=torch.float64))
    s = torch.cat([s, torch.zeros(*s.shape[:2], npad, dtype=torch.float64)], -1)
    if not ids or bool(torch.isinf(s).all()):
        z = torch.zeros(q.shape, dtype=torch.float64).reshape(-1)
        return z, (z, z)
    p = torch.softmax(s, -1)[..., :upto]
    vs = torch.stack([cache[3][layer, max(b, 0)].cpu().double() for b in ids], 1).repeat_interleave(16, 1)[:, :upto]
    codes = torch.stack([cache[1][layer, max(b, 0)].cpu().double() for b in ids]).transpose(0, 1).reshape(nkv, -1, hd)
    loudest = (p * vs[:, None]).amax(-1)
    small = loudest[..., None] * codes[:, :upto].abs().nan_to_num(0.0).sum(1)[:, None]
    return (torch.einsum("grk,gkd->grd", p, x[1]).reshape(-1),
            (torch.einsum("grk,gkd->grd", p, x[1].abs()).reshape(-1), small.reshape(-1)))


def _close(got, want, size, dtype):
    """Elementwise: half a step of the output's type, half a float16 step of every probability
    (float32 queries: two float16 terms, 2^-22), and float32 scores and sums (the exponent of a
    score of magnitude up to 2^5 errs by 2^5 * 2^-22, every sum by some 2^-20).  A float16 step is
    relative only down to 2^-14; below, half a step is 2^-25.  The kernel holds the largest p * vs of a
    tile at 2^8 or above, so a key's weight errs by at most 2^-33 of the largest one, and a sum over
    keys by 2^-33 max(p vs) sum |code|: what is left where the key that takes the whole softmax holds
    a code of exactly 0."""
    size, small = size
    out = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    prob = 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -22
    err = (got.double().cpu() - want).abs()
    limit = out * want.abs() + (prob + 2.0 ** -16) * size + 2.0 ** -33 * small
    assert torch.isfinite(got).all()
    assert (err <= limit * 1.01 + 1e-30).all(), float((err / (limit + 1e-30)).max())


def _tables_for(need, spare, seed):
    NB = sum(need) + spare
    perm = torch.randperm(NB, generator=gen(seed)).tolist()
    tab = np.full((len(need), max(1, max(need))), -1, dtype=np.int32)
    k = 0
    for s, n in enumerate(need):
        tab[s, :n] = perm[k:k + n]
        k += n
    return tab, NB


HEADS = [(32, 8, 128), (8, 8, 64), (8, 1, 128), (6, 2, 32), (16, 1, 64), (28, 4, 128), (32, 4, 64), (5, 1, 32),
         (12, 1, 128)]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,hd", HEADS)
def test_paged_attention_q8(code, dtype, nq, nkv, hd):
    ctx = [1, 16, 17, 0, 70, 333, 15, 600]
    tab, NB = _tables_for([-(-c // 16) for c in ctx], 3, nq)
    cache = _stored(code, NB, nkv, hd, layers=2, seed=nq + hd)
    B = len(ctx)
    wide = torch.randn(B, nq * hd + 24, generator=gen(9)).to(DEV, dtype)
    q = wide[:, : nq * hd]
    order = list(range(B))
    random.Random(1).shuffle(order)
    for pad in (False, True):
        out = torch.full((B, nq * hd + 8), 7.0, dtype=dtype, device=DEV)
        kernels.paged_attention_q8(q, nq, nkv, hd, *cache, 1, torch.from_numpy(tab).to(DEV), i32(order),
                                   i32([ctx[s] for s in order]), pad, 1 / math.sqrt(hd), out=out)
        _lib.check_device_status(DEV, "attention")
        assert (out[:, nq * hd:] == 7.0).all()
        for r, s in enumerate(order):
            want, size = _attend64(q[r], cache, 1, tab[s].tolist(), ctx[s], 1 / math.sqrt(hd),
                                   max(ctx) - ctx[s] if pad else 0)
            _close(out[r, : nq * hd], want, size, dtype)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("B,nq,nkv,hd,lo,hi", [(1, 8, 2, 128, 9001, 9001), (3, 4, 1, 64, 1, 5000),
                                              (200, 8, 8, 32, 1, 150), (64, 32, 8, 128, 100, 1200),
                                              (700, 2, 1, 128, 0, 40)])
def test_paged_attention_q8_splits(code, B, nq, nkv, hd, lo, hi):
    """Long, many and ragged rows: however the work is split, every row is its own softmax."""
    rng = random.Random(B)
    ctx = [rng.randint(lo, hi) for _ in range(B)]
    tab, NB = _tables_for([-(-c // 16) for c in ctx], 1, B)
    cache = _stored(code, NB, nkv, hd, seed=B)
    q = torch.randn(B, nq * hd, generator=gen(B)).to(DEV, torch.bfloat16)
    out = kernels.paged_attention_q8(q, nq, nkv, hd, *cache, 0, torch.from_numpy(tab).to(DEV), None, i32(ctx), False,
                                     1 / math.sqrt(hd))
    _lib.check_device_status(DEV, "attention")
    for r in sorted(rng.sample(range(B), min(B, 40))):
        want, size = _attend64(q[r], cache, 0, tab[r].tolist(), ctx[r], 1 / math.sqrt(hd))
        _close(out[r], want, size, torch.bfloat16)
    again = kernels.paged_attention_q8(q, nq, nkv, hd, *cache, 0, torch.from_numpy(tab).to(DEV), None, i32(ctx), False,
                                       1 / math.sqrt(hd))
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_paged_attention_q8_wide_ranges(dtype):
    """Scales that differ by 2^40 between blocks, zero scales, large and tiny queries: the
    statistics hold, and a loud block does not drown a quiet one that the softmax prefers."""
    nq, nkv, hd, ctx = 4, 2, 64, 160
    tab, NB = _tables_for([10, 10, 10, 10], 2, 1)
    cache = _stored("int8", NB, nkv, hd, seed=4)
    cache[3] *= torch.exp2(torch.randint(-20, 20, cache[3].shape, generator=gen(5)).float()).to(DEV)
    cache[3][0, tab[1, 3]] = 0
    cache[2][0, tab[2, 4]] = 0
    q = torch.randn(4, nq * hd, generator=gen(6))
    q[0] *= 2.0 ** -60
    q[1] *= 4
    q[2, :hd] = 0
    q[3] *= torch.exp2(torch.randint(-30, 3, q[3].shape, generator=gen(7)).float())
    q = q.to(DEV, dtype)
    out = kernels.paged_attention_q8(q, nq, nkv, hd, *cache, 0, torch.from_numpy(tab).to(DEV), None, i32([ctx] * 4),
                                     False, 1 / math.sqrt(hd))
    for r in range(4):
        want, size = _attend64(q[r], cache, 0, tab[r].tolist(), ctx, 1 / math.sqrt(hd))
        _close(out[r], want, size, dtype)


@pytest.mark.parametrize("lens,ctx0", [([90, 40], [100, 0]), ([3, 2], [100, 7])])
@pytest.mark.parametrize("nq,nkv", [(4, 2), (6, 2)])
def test_prefill_attention_q8_wide_ranges(nq, nkv, lens, ctx0):
    """The same for the kernels of many tokens per sequence."""
    hd = 128
    tab, NB = _tables_for([-(-(c + n) // 16) for c, n in zip(ctx0, lens)], 2, 1)
    cache = _stored("int8", NB, nkv, hd, seed=4)
    cache[3] *= torch.exp2(torch.randint(-20, 20, cache[3].shape, generator=gen(5)).float()).to(DEV)
    for j in (0, 1):
        cache[3][0, tab[0, j]] = 0
    cache[3][0, tab[1, 0]] = 0
    cache[2][0, tab[0, 2]] = 0
    q = torch.randn(sum(lens), nq * hd, generator=gen(6))
    q[::3] *= 6
    q[1::5] *= 2.0 ** -60
    q = q.to(DEV, torch.bfloat16)
    start = [0, lens[0], sum(lens)]
    out = kernels.prefill_attention_q8(q, nq, nkv, hd, *cache, 0, torch.from_numpy(tab).to(DEV), i32(start), 2,
                                       1 / math.sqrt(hd), seq_ctx0=i32(ctx0))
    _lib.check_device_status(DEV, "prefill")
    for s, n in enumerate(lens):
        for i in range(n):
            r = start[s] + i
            want, size = _attend64(q[r], cache, 0, tab[s].tolist(), ctx0[s] + i + 1, 1 / math.sqrt(hd))
            _close(out[r], want, size, torch.bfloat16)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_attention_q8_ignores_what_lies_behind_the_context(code):
    """Codes (NaN ones too) behind the context, blocks behind it and their scales change nothing."""
    nq, nkv, hd = 8, 2, 64
    ctx = [5, 21, 40]
    tab, NB = _tables_for([4, 4, 4], 1, 2)
    cache = _stored(code, NB, nkv, hd, seed=8)
    q = torch.randn(3, nq * hd, generator=gen(3)).to(DEV, torch.bfloat16)
    t = torch.from_numpy(tab).to(DEV)
    first = kernels.paged_attention_q8(q, nq, nkv, hd, *cache, 0, t, None, i32(ctx), False, 0.1)
    start, c0 = i32([0, 1, 2, 3]), i32([c - 1 for c in ctx])
    pre = kernels.prefill_attention_q8(q, nq, nkv, hd, *cache, 0, t, start, 3, 0.1, seq_ctx0=c0)
    for r, c in enumerate(ctx):
        for j in range(4):
            b = int(tab[r, j])
            keep = max(0, min(16, c - 16 * j))
            for x in (cache[0], cache[1]):
                x[0, b].view(torch.uint8)[:, keep:] = 0x7f  # e4m3: NaN
            if keep == 0:
                cache[2][0, b] = float("nan")
                cache[3][0, b] = float("inf")
    t2 = t.clone()
    t2[0, 1:] = -5
    again = kernels.paged_attention_q8(q, nq, nkv, hd, *cache, 0, t2, None, i32(ctx), False, 0.1)
    assert torch.equal(first, again)
    assert torch.equal(pre, kernels.prefill_attention_q8(q, nq, nkv, hd, *cache, 0, t2, start, 3, 0.1, seq_ctx0=c0))
    _lib.check_device_status(DEV, "attention")
    # a tile poisoned by a value that was not finite reaches the rows that see it, and no others
    cache[2][0, int(tab[1, 0])] = float("nan")
    out = kernels.paged_attention_q8(q, nq, nkv, hd, *cache, 0, t2, None, i32(ctx), False, 0.1)
    assert torch.isnan(out[1]).all() and torch.equal(out[0], first[0]) and torch.equal(out[2], first[2])


def test_attention_q8_skips_and_reports_bad_pages():
    nq, nkv, hd = 8, 2, 128
    ctx = [100, 300, 64]
    tab, NB = _tables_for([-(-c // 16) for c in ctx], 2, 2)
    cache = _stored("int8", NB, nkv, hd, seed=8)
    q = torch.randn(3, nq * hd, generator=gen(3)).to(DEV, torch.bfloat16)
    bad = tab.copy()
    bad[0, 3], bad[1, 0], bad[1, 7] = NB, -1, 1 << 30
    clean = np.where((bad < 0) | (bad >= NB), -1, bad)
    scale = 1 / math.sqrt(hd)
    out = kernels.paged_attention_q8(q, nq, nkv, hd, *cache, 0, torch.from_numpy(bad).to(DEV), None, i32(ctx), False, scale)
    with pytest.raises(IndexError):
        _lib.check_device_status(DEV, "attention")
    pre = kernels.prefill_attention_q8(q, nq, nkv, hd, *cache, 0, torch.from_numpy(bad).to(DEV), i32([0, 1, 2, 3]), 3,
                                       scale, seq_ctx0=i32([c - 1 for c in ctx]))
    with pytest.raises(IndexError):
        _lib.check_device_status(DEV, "prefill")
    for r in range(3):
        want, size = _attend64(q[r], cache, 0, clean[r].tolist(), ctx[r], scale)
        _close(out[r], want, size, torch.bfloat16)
        _close(pre[r], want, size, torch.bfloat16)
    # a context longer than its table row sees the row's keys; a table row that is not there, none
    t = torch.from_numpy(tab).to(DEV)
    out = kernels.paged_attention_q8(q[:2], nq, nkv, hd, *cache, 0, t[:2, :4].contiguous(), i32([1, 2]),
                                     i32([300, 64]), False, scale)
    with pytest.raises(IndexError):
        _lib.check_device_status(DEV, "attention")
    want, size = _attend64(q[0], cache, 0, tab[1].tolist(), 64, scale)
    _close(out[0], want, size, torch.bfloat16)
    assert (out[1] == 0).all()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,hd", HEADS)
def test_prefill_attention_q8(code, dtype, nq, nkv, hd):
    lens = [1, 16, 0, 17, 70, 5, 130, 33]
    ctx0 = [0, 0, 3, 5, 0, 300, 33, 64]
    tab, NB = _tables_for([-(-(c + n) // 16) for c, n in zip(ctx0, lens)], 3, nq)
    cache = _stored(code, NB, nkv, hd, layers=2, seed=nq + hd)
    T = sum(lens)
    q = torch.randn(T + 2, nq * hd + 16, generator=gen(9)).to(DEV, dtype)[:, : nq * hd]
    start = np.concatenate([[0], np.cumsum(lens)])
    out = torch.full((T + 2, nq * hd), 7.0, dtype=dtype, device=DEV)
    kernels.prefill_attention_q8(q, nq, nkv, hd, *cache, 1, torch.from_numpy(tab).to(DEV), i32(start.tolist()),
                                 len(lens), 1 / math.sqrt(hd), seq_ctx0=i32(ctx0), out=out)
    _lib.check_device_status(DEV, "prefill")
    assert (out[T:] == 7.0).all()  # rows behind the last sequence
    for s, n in enumerate(lens):
        for i in sorted({0, 1, 15, 16, n // 2, n - 1} & set(range(n))):
            r = int(start[s]) + i
            want, size = _attend64(q[r], cache, 1, tab[s].tolist(), ctx0[s] + i + 1, 1 / math.sqrt(hd))
            _close(out[r], want, size, dtype)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("nq,nkv,lens,ctx0", [(32, 8, [1024, 700, 65], [0, 0, 2000]), (8, 1, [300] * 5, [17] * 5),
                                             (4, 4, [513], [0]), (8, 4, [129, 1, 640], [1, 900, 31])])
def test_prefill_attention_q8_long(code, nq, nkv, lens, ctx0):
    hd = 128
    tab, NB = _tables_for([-(-(c + n) // 16) for c, n in zip(ctx0, lens)], 3, nq)
    cache = _stored(code, NB, nkv, hd, seed=nq + hd)
    T = sum(lens)
    q = torch.randn(T, nq * hd, generator=gen(9)).to(DEV, torch.bfloat16)
    start = np.concatenate([[0], np.cumsum(lens)])
    out = kernels.prefill_attention_q8(q, nq, nkv, hd, *cache, 0, torch.from_numpy(tab).to(DEV), i32(start.tolist()),
                                       len(lens), 1 / math.sqrt(hd), seq_ctx0=i32(ctx0))
    _lib.check_device_status(DEV, "prefill")
    for s, n in enumerate(lens):
        for i in sorted({0, 31, 32, 63, 64, 127, 128, n // 2, n - 2, n - 1} & set(range(n))):
            r = int(start[s]) + i
            want, size = _attend64(q[r], cache, 0, tab[s].tolist(), ctx0[s] + i + 1, 1 / math.sqrt(hd))
            _close(out[r], want, size, torch.bfloat16)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("nq,nkv", [(16, 16), (16, 8), (16, 4), (16, 2), (15, 5), (20, 4), (18, 3), (14, 2), (24, 2),
                                    (32, 2)])
def test_prefill_attention_q8_many_rows(code, nq, nkv):
    """Enough rows for the tcgen05 kernel at every number of heads to a kv head, with what may go wrong in it: an
    empty sequence, scales that differ by 2^40 and are 0, pages outside the pool, NaN codes behind the context,
    padded q rows, and rows behind the last sequence."""
    hd, lens, ctx0 = 128, [200, 0, 250], [40, 0, 7]
    tab, NB = _tables_for([-(-(c + n) // 16) for c, n in zip(ctx0, lens)], 2, 1)
    cache = _stored(code, NB, nkv, hd, seed=4)
    cache[3] *= torch.exp2(torch.randint(-20, 20, cache[3].shape, generator=gen(5)).float()).to(DEV)
    for j in (0, 1):
        cache[3][0, tab[0, j]] = 0
    cache[2][0, tab[0, 2]] = 0
    for s in (0, 2):
        last = ctx0[s] + lens[s] - 1
        for x in (cache[0], cache[1]):
            x[0, int(tab[s, last // 16])].view(torch.uint8)[:, last % 16 + 1:] = 0x7f  # e4m3: NaN
    T = sum(lens)
    q = torch.randn(T + 3, nq * hd + 8, generator=gen(6))
    q[::3] *= 6
    q[1::5] *= 2.0 ** -60
    q = q.to(DEV, torch.bfloat16)[:, : nq * hd]
    start = np.concatenate([[0], np.cumsum(lens)])
    bad = tab.copy()
    bad[0, 5], bad[2, 1], bad[2, 9] = NB, -1, 1 << 30
    clean = np.where((bad < 0) | (bad >= NB), -1, bad)
    for t, pages in ((tab, tab), (bad, clean)):
        out = torch.full((T + 3, nq * hd), 7.0, dtype=torch.bfloat16, device=DEV)
        kernels.prefill_attention_q8(q, nq, nkv, hd, *cache, 0, torch.from_numpy(t).to(DEV), i32(start.tolist()), 3,
                                     1 / math.sqrt(hd), seq_ctx0=i32(ctx0), out=out)
        if t is bad:
            with pytest.raises(IndexError):
                _lib.check_device_status(DEV, "prefill")
        _lib.check_device_status(DEV, "prefill")
        assert (out[T:] == 7.0).all()
        for s, n in enumerate(lens):
            for i in sorted({0, 15, 16, 31, 63, 64, 127, 128, n // 2, n - 1} & set(range(n))):
                r = int(start[s]) + i
                want, size = _attend64(q[r], cache, 0, pages[s].tolist(), ctx0[s] + i + 1, 1 / math.sqrt(hd))
                _close(out[r], want, size, torch.bfloat16)


@pytest.mark.parametrize("nq,nkv,n,longest", [(8, 1, 300, 32), (4, 2, 700, 6)])
def test_prefill_attention_q8_many_sequences(nq, nkv, n, longest):
    """More sequences than a CTA keeps the lengths of (192 in the tcgen05 kernel, 256 groups in the mma one), many of
    them empty."""
    hd = 128
    lens = torch.randint(0, longest, (n,), generator=gen(1)).tolist()
    ctx0 = torch.randint(0, 40, (n,), generator=gen(2)).tolist()
    lens[0] = lens[-1] = 0
    tab, NB = _tables_for([-(-(c + m) // 16) for c, m in zip(ctx0, lens)], 3, nq)
    cache = _stored("int8", NB, nkv, hd, seed=nq)
    T = sum(lens)
    q = torch.randn(T, nq * hd, generator=gen(9)).to(DEV, torch.bfloat16)
    start = np.concatenate([[0], np.cumsum(lens)])
    out = kernels.prefill_attention_q8(q, nq, nkv, hd, *cache, 0, torch.from_numpy(tab).to(DEV), i32(start.tolist()),
                                       n, 1 / math.sqrt(hd), seq_ctx0=i32(ctx0))
    _lib.check_device_status(DEV, "prefill")
    for s in list(range(0, n, 37)) + [n - 2, n - 1]:
        for i in sorted({0, lens[s] - 1} & set(range(lens[s]))):
            r = int(start[s]) + i
            want, size = _attend64(q[r], cache, 0, tab[s].tolist(), ctx0[s] + i + 1, 1 / math.sqrt(hd))
            _close(out[r], want, size, torch.bfloat16)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("nkv,n", [(16, 400), (2, 60)])
def test_a_value_that_is_not_finite_reaches_no_row_before_its_block(code, nkv, n):
    """Written and read in one call: tcgen05 tiles (400 tokens, 16 heads) and mma tiles hold rows of several
    blocks, of which those before the poisoned one keep their bits."""
    hd, at = 128, 37
    rope = RotaryEmbedding(hd, 512, 10000.0, DEV)
    outs = []
    for x in (1.0, float("inf"), float("nan")):
        qkv, pos, row, tab, NB = _step([n], [0], nkv, nkv, hd, torch.bfloat16, 2)
        qkv.view(n, 3 * nkv, hd)[at, nkv:, 5] = x
        cache = _caches(code, NB, nkv, hd, seed=3)
        q = _write(qkv, nkv, nkv, hd, None, pos, row, tab, rope, cache)
        outs.append(kernels.prefill_attention_q8(q, nkv, nkv, hd, *cache, 0, tab, i32([0, n]), 1, 0.1))
        _lib.check_device_status(DEV, "poison")
    assert torch.isfinite(outs[0]).all()
    for out in outs[1:]:
        assert torch.equal(out[:32], outs[0][:32]) and torch.isnan(out[32:]).all()


def test_attention_q8_refusals():
    nq, nkv, hd = 4, 2, 64
    cache = _stored("int8", 4, nkv, hd)
    q = torch.randn(2, nq * hd, device=DEV, dtype=torch.bfloat16)
    t, ctx = i32([[0], [1]]), i32([3, 4])

    def call(q=q, nq=nq, nkv=nkv, hd=hd, c=cache, layer=0, t=t, ctx=ctx, idx=None, out=None):
        return kernels.paged_attention_q8(q, nq, nkv, hd, *c, layer, t, idx, ctx, False, 0.1, out=out)

    call()
    bad = [dict(q=q.half()), dict(q=q.cpu()), dict(q=q[:, :-8]), dict(q=q[:, 4:]), dict(nq=3), dict(nkv=1),
           dict(hd=32), dict(c=[cache[0].float()] + cache[1:]), dict(c=[cache[0][:, :3]] + cache[1:]),
           dict(c=cache[:2] + [cache[2].double(), cache[3]]), dict(c=cache[:3] + [cache[3][:, :2].contiguous()]),
           dict(layer=1), dict(t=t.long()), dict(t=t[:1]), dict(ctx=ctx.long()), dict(ctx=ctx[:1]),
           dict(idx=ctx.long()), dict(out=q.float()), dict(out=q[:1])]
    for kw in bad:
        with pytest.raises((_lib.B2Error, IndexError)):
            call(**kw)
    big = _stored("int8", 4, 1, 64)
    with pytest.raises(_lib.B2Error, match="nq/nkv"):
        kernels.paged_attention_q8(torch.zeros(2, 17 * 64, device=DEV), 17, 1, 64, *big, 0, t, None, ctx, False, 0.1)
    wide = [torch.zeros(1, 4, 2, 32, 64, dtype=torch.int8, device=DEV)] * 2 + cache[2:]
    with pytest.raises(_lib.B2Error, match="block_size"):
        call(c=wide)
    with pytest.raises(_lib.B2Error, match="table rows"):
        kernels.prefill_attention_q8(q, nq, nkv, hd, *cache, 0, t, i32([0, 1, 1, 2]), 3, 0.1)
    assert call(q=q[:0], ctx=ctx[:0]).shape == (0, nq * hd)
    _lib.check_device_status(DEV, "refusals")


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_a_serving_run(code):
    """Admit prompts, prefill them in two chunks, draft, roll back and decode: tables, maps, cache
    and attention together, against float64 attention over what was written."""
    nq, nkv, hd, bs, n, width = 8, 2, 128, 16, 5, 12
    pool = 40
    tables, lens, ring, state, host = _device_tables(n, width, pool, bs, 33, 3)
    rope = RotaryEmbedding(hd, 256, 10000.0, DEV)
    w = (1 + 0.2 * torch.randn(hd, generator=gen(1))).to(DEV)
    cache = _caches(code, pool, nkv, hd)
    scale = 1 / math.sqrt(hd)
    full = [[] for _ in range(n)]  # exact keys and values as they were given
    steps = [("new", [40, 0, 17, 1, 33]), ("new", [25, 16, 0, 3, 33]), ("new", [1, 1, 1, 1, 1]), ("new", [4, 4, 0, 4, 4]),
             ("keep", [67, 18, 18, 6, 200]), ("keep", [67, 0, 18, 6, 200]), ("new", [1, 30, 1, 1, 1])]
    for k, (what, vals) in enumerate(steps):
        if what == "keep":
            kernels.block_tables_truncate(tables, lens, i32(vals), bs, ring, state)
            host.truncate(vals)
            full = [f[:m] for f, m in zip(full, vals)]
            continue
        T = sum(vals)
        ctx0 = lens.clone()
        m = kernels.block_tables_extend(tables, lens, i32(vals), T, bs, ring, state)
        host.extend(vals)
        qkv = torch.randn(T, (nq + 2 * nkv) * hd, generator=gen(50 + k)).to(DEV, torch.bfloat16)
        q = _write(qkv, nq, nkv, hd, w, m.positions, m.table_index, tables, rope, cache)
        if max(vals) == 1:
            out = kernels.paged_attention_q8(q, nq, nkv, hd, *cache, 0, tables, m.table_index, m.ctx_lens, False, scale)
        else:
            out = kernels.prefill_attention_q8(q, nq, nkv, hd, *cache, 0, tables, m.seq_start, n, scale, seq_ctx0=ctx0)
        _lib.check_device_status(DEV, "step")
        x = qkv.view(T, -1, hd)
        kx = _norm_rotate64(x[:, nq:nq + nkv], w, 1e-5, rope.cos_cached[m.positions], rope.sin_cached[m.positions]).cpu()
        vx = x[:, nq + nkv:].double().cpu()
        rows, pos = m.table_index.tolist(), m.positions.tolist()
        for t in range(T):
            full[rows[t]].append((kx[t], vx[t]))
        for t in range(0, T, 3):
            s = rows[t]
            want, size = _attend64(q[t], cache, 0, host.tables[s], pos[t] + 1, scale)
            _close(out[t], want, size, torch.bfloat16)
            # and near the attention over the values that were never rounded to 8 bits
            ks = torch.stack([a for a, _ in full[s][: pos[t] + 1]], 1)
            vs = torch.stack([b for _, b in full[s][: pos[t] + 1]], 1)
            p = torch.softmax(torch.einsum("grd,gkd->grk", q[t].double().cpu().view(nkv, -1, hd), ks) * scale, -1)
            exact = torch.einsum("grk,gkd->grd", p, vs).reshape(-1)
            assert float((out[t].double().cpu() - exact).norm() / exact.norm()) < (0.04 if code == "int8" else 0.12)


def test_streams_and_graphs_do_not_share_scratch():
    """Two calls at once on two streams, and two captured graphs replayed at once, against the same calls alone."""
    nq, nkv, hd = 8, 2, 128
    cases = []
    for k, ctx in enumerate(([4000, 3], [900, 2500, 1])):
        tab, NB = _tables_for([-(-c // 16) for c in ctx], 1, k)
        cache = _stored("int8", NB, nkv, hd, seed=k)
        q = torch.randn(len(ctx), nq * hd, generator=gen(k)).to(DEV, torch.bfloat16)
        cases.append((q, cache, torch.from_numpy(tab).to(DEV), i32(ctx)))

    def call(c):
        q, cache, t, ctx = c
        return kernels.paged_attention_q8(q, nq, nkv, hd, *cache, 0, t, None, ctx, False, 0.1)

    want = [call(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(c))
        graphs.append(g)
    for _ in range(20):
        got = []
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(call(c))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
