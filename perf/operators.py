"""The serving operators around the 8-bit paged KV cache: what is measured and against which plain form.

Three groups of entry points of ``pythonintern_b200.kernels``, in the order a step runs them:

* ``block_tables_extend`` / ``block_tables_truncate``: block tables and slot maps built on the
  GPU from request lengths;
* ``qk_norm_rope_kv_write`` / ``qk_norm_rope_kv_write_q8`` (and ``kv_read_q8``, which reads tiles
  back): per-head RMS norms of queries and keys, the rotation and the paged cache write in one
  pass, into a cache of the model's type or of 8 bits with a scale per block and head;
* ``paged_attention_q8`` / ``prefill_attention_q8``: attention over the 8-bit cache, one query
  token per row or many per sequence.

``listed()`` names the cases, ``draw()`` makes more of the same ranges, ``prepare()`` builds the
inputs, ``run()`` makes one pass: the plain torch form where ``own`` is false, the framework's
entry points where it is true.  ``exact()`` restates the definition in 64 bits.

Layouts.  8-bit caches: [layers, blocks, kv heads, 16 tokens, head_dim], int8 or float8_e4m3fn;
scales: float32 [layers, blocks, kv heads].  Caches of the model's type: [layers, blocks, 16
tokens, kv heads, head_dim].  Every cache here has one layer.
"""

import math
import random

import torch

own = False

BLOCK = 16
EPS = 1e-5
TOP = {"int8": 127.0, "e4m3": 448.0}      # largest code
TINY = 2.0 ** -126                        # a scale below this stands for a tile of zeros
MAX_POS = 16384                           # rows of the cos/sin tables

# (q heads, kv heads, head_dim)
HEADS = [(32, 8, 128), (32, 4, 64), (8, 2, 32), (8, 8, 64), (8, 1, 128), (12, 4, 64), (28, 4, 128), (16, 1, 64)]


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one speculative step of a decode batch: four drafted tokens per request, all refused
        {"name": "tables_draft_128", "op": "tables", "requests": 128, "ctx_lo": 1, "ctx_hi": 2000, "new_lo": 4,
         "new_hi": 4, "mix": 1},
        # a batch of prompts is admitted and leaves again
        {"name": "tables_admit_16x1024", "op": "tables", "requests": 16, "ctx_lo": 0, "ctx_hi": 0, "new_lo": 1024,
         "new_hi": 1024, "mix": 2},
        # many requests of every length, idle ones among them
        {"name": "tables_ragged_2048", "op": "tables", "requests": 2048, "ctx_lo": 0, "ctx_hi": 4000, "new_lo": 0,
         "new_hi": 200, "mix": 3},
        # the smallest decode step: latency
        {"name": "write_bf16_decode_8", "op": "write", "dtype": "bfloat16", "nq": 32, "nkv": 8, "hd": 128,
         "requests": 8, "ctx_lo": 100, "ctx_hi": 2000, "new_lo": 1, "new_hi": 1, "mix": 4},
        # a full decode batch, tokens landing inside blocks that hold earlier ones
        {"name": "write_int8_decode_128", "op": "write_q8", "dtype": "bfloat16", "code": "int8", "nq": 32, "nkv": 8,
         "hd": 128, "requests": 128, "ctx_lo": 1, "ctx_hi": 2047, "new_lo": 1, "new_hi": 1, "mix": 5},
        # a batched prefill step
        {"name": "write_bf16_prefill_16x1024", "op": "write", "dtype": "bfloat16", "nq": 32, "nkv": 8, "hd": 128,
         "requests": 16, "ctx_lo": 0, "ctx_hi": 0, "new_lo": 1024, "new_hi": 1024, "mix": 6},
        # chunks of prompts of odd lengths that go on behind cached ones
        {"name": "write_e4m3_prefill_ragged", "op": "write_q8", "dtype": "bfloat16", "code": "e4m3", "nq": 32,
         "nkv": 4, "hd": 64, "requests": 37, "ctx_lo": 0, "ctx_hi": 500, "new_lo": 1, "new_hi": 511, "mix": 7},
        # one user, a long context: latency and the split over the context
        {"name": "decode_int8_1x8192", "op": "decode_q8", "dtype": "bfloat16", "code": "int8", "nq": 32, "nkv": 8,
         "hd": 128, "requests": 1, "ctx_lo": 8192, "ctx_hi": 8192, "mix": 8},
        # the ordinary decode batch: bandwidth
        {"name": "decode_int8_128x2048", "op": "decode_q8", "dtype": "bfloat16", "code": "int8", "nq": 32, "nkv": 8,
         "hd": 128, "requests": 128, "ctx_lo": 2048, "ctx_hi": 2048, "mix": 9},
        # a batch of very different contexts, an empty row possible, heads of 64
        {"name": "decode_e4m3_ragged_61", "op": "decode_q8", "dtype": "bfloat16", "code": "e4m3", "nq": 32, "nkv": 4,
         "hd": 64, "requests": 61, "ctx_lo": 0, "ctx_hi": 8191, "mix": 10},
        # drafted tokens checked against long contexts
        {"name": "prefill_e4m3_draft_48x5", "op": "prefill_q8", "dtype": "bfloat16", "code": "e4m3", "nq": 32,
         "nkv": 8, "hd": 128, "requests": 48, "ctx_lo": 500, "ctx_hi": 4000, "new_lo": 5, "new_hi": 5, "mix": 11},
        # a batched prefill step
        {"name": "prefill_int8_16x1024", "op": "prefill_q8", "dtype": "bfloat16", "code": "int8", "nq": 32, "nkv": 8,
         "hd": 128, "requests": 16, "ctx_lo": 0, "ctx_hi": 0, "new_lo": 1024, "new_hi": 1024, "mix": 12},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 0.2)))))


def draw(rng):
    op = rng.choice(["tables", "write", "write_q8", "decode_q8", "prefill_q8"])
    mix = rng.randrange(1 << 20)
    if op == "tables":
        requests = _log_int(rng, 1, 2048)
        if rng.random() < 0.5:
            ctx_hi, new_lo, new_hi = rng.randint(1, 4000), 1, rng.randint(1, 8)
        else:
            ctx_hi, new_lo, new_hi = rng.choice([0, rng.randint(1, 4000)]), 0, _log_int(rng, 8, min(1024, 400000 // requests))
        return {"op": op, "requests": requests, "ctx_lo": 0, "ctx_hi": ctx_hi, "new_lo": new_lo, "new_hi": new_hi, "mix": mix}
    nq, nkv, hd = rng.choice(HEADS)
    case = {"op": op, "dtype": "bfloat16" if op == "prefill_q8" or rng.random() < 0.8 else "float32"}
    if op != "write":
        case["code"] = rng.choice(["int8", "e4m3"])
    case |= {"nq": nq, "nkv": nkv, "hd": hd}
    if op == "decode_q8":
        requests = _log_int(rng, 1, 256)
        most = min(16000, 128 * 2048 * 1024 // (requests * nkv * hd))
        hi = _log_int(rng, 16, most)
        return case | {"requests": requests, "ctx_lo": rng.choice([0, 1, hi // 2, hi]), "ctx_hi": hi, "mix": mix}
    if op == "prefill_q8":
        requests = _log_int(rng, 1, 64)
        new_hi = _log_int(rng, 1, min(2048, 16384 // requests))
        most = 16 * 1024 * 1024 * 32 // (requests * new_hi * nq)  # keys a padded row may see
        ctx_hi = rng.choice([0, _log_int(rng, 1, max(1, min(8000, most - new_hi)))])
        return case | {"requests": requests, "ctx_lo": 0, "ctx_hi": max(0, min(ctx_hi, most - new_hi)),
                       "new_lo": rng.choice([1, new_hi]), "new_hi": new_hi, "mix": mix}
    decode = rng.random() < 0.5
    requests = _log_int(rng, 1, 256 if decode else 64)
    new_hi = 1 if decode else _log_int(rng, 2, min(4096, 16384 // requests))
    ctx_hi = rng.choice([0, rng.randint(1, 2047)])
    return case | {"requests": requests, "ctx_lo": 0, "ctx_hi": ctx_hi, "new_lo": rng.choice([1, new_hi]),
                   "new_hi": new_hi, "mix": mix}


def _lengths(case):
    """(cached tokens, new tokens) of each request: of the case alone, so every seed has the same shapes."""
    r = random.Random(case["mix"])
    n = case["requests"]
    ctx = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(n)]
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(n)] if "new_hi" in case else [0] * n
    return ctx, new


def _blocks(tokens):
    return -(-tokens // BLOCK)


# --------------------------------------------------------------------------- inputs
def _dtype(case):
    return {"bfloat16": torch.bfloat16, "float32": torch.float32}[case["dtype"]]


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _tables(lens, gen, spare):
    """Block tables over a permuted pool, -1 behind each row's last block: (tables, pool size, ids not in use)."""
    need = [_blocks(n) for n in lens]
    total = sum(need)
    perm = torch.randperm(total + spare, generator=gen, device="cuda").to(torch.int32)
    width = max(1, max(need))
    need_t = _ints(need, torch.int64)
    start = torch.cumsum(need_t, 0) - need_t
    col = torch.arange(width, device="cuda")
    at = (start[:, None] + col).clamp_max(total + spare - 1)
    tables = torch.where(col < need_t[:, None], perm[at], torch.full_like(perm[at], -1))
    return tables.contiguous(), total + spare, perm[total:].contiguous()


def _stored(blocks, nkv, hd, code, gen):
    """An 8-bit cache in use: normal values, some heads louder than others, a scale for each tile."""
    x = torch.randn(blocks, nkv, BLOCK, hd, generator=gen, device="cuda")
    loud = torch.rand(blocks, nkv, 1, 1, generator=gen, device="cuda").mul_(1.5).add_(0.5)
    scale = x.abs().amax((2, 3), keepdim=True).mul_(1.0 / TOP[code])
    x.div_(scale)
    codes = x.round_().to(torch.int8) if code == "int8" else x.clamp_(-448, 448).to(torch.float8_e4m3fn)
    return codes[None], (scale * loud).reshape(1, blocks, nkv)


def _rotation(hd):
    inv = 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    angle = torch.arange(MAX_POS, dtype=torch.float64, device="cuda")[:, None] * inv
    angle = torch.cat([angle, angle], dim=1)
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    ctx, new = _lengths(case)
    if case["op"] == "tables":
        width = max(1, max(_blocks(c + n) for c, n in zip(ctx, new)))
        taken = sum(_blocks(c + n) - _blocks(c) for c, n in zip(ctx, new))
        held, pool, free = _tables(ctx, gen, taken + 64)
        tables = torch.full((len(ctx), width), -1, dtype=torch.int32, device="cuda")
        tables[:, :held.shape[1]] = held[:, :width]
        head = int(torch.randint(0, pool, (1,), generator=gen, device="cuda"))
        ring = torch.full((pool,), -1, dtype=torch.int32, device="cuda")
        ring[(head + torch.arange(free.numel(), device="cuda")) % pool] = free
        return {"case": case, "tables": tables, "lens": _ints(ctx), "new": _ints(new), "keep": _ints(ctx),
                "ring": ring, "free": _ints([head, free.numel(), 0, 0]), "tokens": sum(new)}
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    after = [c + n for c, n in zip(ctx, new)]
    tables, pool, _ = _tables(after, gen, 5)
    dtype = _dtype(case)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    state = {"case": case, "tables": tables, "tokens": start[-1], "width": tables.shape[1], "most": max(new),
             "ctx0": _ints(ctx), "seq_start": _ints(start), "ctx_lens": _ints(ctx)}
    if "code" in case:
        state["k"], state["ks"] = _stored(pool, nkv, hd, case["code"], gen)
        state["v"], state["vs"] = _stored(pool, nkv, hd, case["code"], gen)
    if case["op"] == "decode_q8":
        state["q"] = torch.randn(len(ctx), nq * hd, generator=gen, device="cuda").to(dtype)
        return state
    if case["op"] == "prefill_q8":
        state["q"] = torch.randn(start[-1], nq * hd, generator=gen, device="cuda").to(dtype)
        return state
    row = torch.repeat_interleave(torch.arange(len(new), device="cuda"), _ints(new, torch.int64))
    pos = torch.arange(start[-1], device="cuda") - state["seq_start"][row] + state["ctx0"][row]
    state["pos"], state["row"] = pos.to(torch.int64), row.to(torch.int32)
    state["qkv"] = torch.randn(start[-1], (nq + 2 * nkv) * hd, generator=gen, device="cuda").mul_(2.0).to(dtype)
    state["wq"] = 1.0 + 0.2 * torch.randn(hd, generator=gen, device="cuda")
    state["wk"] = 1.0 + 0.2 * torch.randn(hd, generator=gen, device="cuda")
    state["cos"], state["sin"] = _rotation(hd)
    # the blocks that the step's tokens land in, request by request
    cols = [j for c, n in zip(ctx, new) for j in range(c // BLOCK, _blocks(c + n))]
    rows = [s for s, (c, n) in enumerate(zip(ctx, new)) for j in range(c // BLOCK, _blocks(c + n))]
    state["touched"] = tables[_ints(rows, torch.int64), _ints(cols, torch.int64)].contiguous()
    if case["op"] == "write":
        state["k"] = torch.randn(1, pool, BLOCK, nkv, hd, generator=gen, device="cuda").to(dtype)
        state["v"] = torch.randn(1, pool, BLOCK, nkv, hd, generator=gen, device="cuda").to(dtype)
    return state


# --------------------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"tables": _own_tables, "write": _own_write, "write_q8": _own_write_q8, "decode_q8": _own_decode,
                "prefill_q8": _own_prefill}[op](state)
    return {"tables": _plain_tables, "write": _plain_write, "write_q8": _plain_write_q8, "decode_q8": _plain_decode,
            "prefill_q8": _plain_prefill}[op](state)


def _own_tables(st):
    from pythonintern_b200 import kernels
    m = kernels.block_tables_extend(st["tables"], st["lens"], st["new"], st["tokens"], BLOCK, st["ring"], st["free"])
    kernels.block_tables_truncate(st["tables"], st["lens"], st["keep"], BLOCK, st["ring"], st["free"])
    return [m.seq_start, m.positions, m.table_index, m.slots, m.ctx_lens, m.last_rows, st["tables"], st["lens"],
            st["ring"], st["free"]]


def _own_write(st):
    from pythonintern_b200 import kernels
    c = st["case"]
    q = torch.empty(st["tokens"], c["nq"] * c["hd"], dtype=st["qkv"].dtype, device=st["qkv"].device)
    kernels.qk_norm_rope_kv_write(st["qkv"], c["nq"], c["nkv"], c["hd"], st["wq"], st["wk"], EPS, st["pos"], None,
                                  st["row"], st["tables"], st["cos"], st["sin"], q, st["k"], st["v"], 0)
    return [q, st["k"], st["v"]]


def _own_write_q8(st):
    from pythonintern_b200 import kernels
    c = st["case"]
    q = torch.empty(st["tokens"], c["nq"] * c["hd"], dtype=st["qkv"].dtype, device=st["qkv"].device)
    kernels.qk_norm_rope_kv_write_q8(st["qkv"], c["nq"], c["nkv"], c["hd"], st["wq"], st["wk"], EPS, st["pos"], None,
                                     st["row"], st["tables"], st["cos"], st["sin"], q, st["k"], st["v"], st["ks"],
                                     st["vs"], 0)
    k, v = kernels.kv_read_q8(st["k"], st["v"], st["ks"], st["vs"], 0, st["touched"], torch.bfloat16)
    return [q, k, v, st["ks"], st["vs"]]


def _own_decode(st):
    from pythonintern_b200 import kernels
    c = st["case"]
    return [kernels.paged_attention_q8(st["q"], c["nq"], c["nkv"], c["hd"], st["k"], st["v"], st["ks"], st["vs"], 0,
                                       st["tables"], None, st["ctx_lens"], False, 1.0 / math.sqrt(c["hd"]))]


def _own_prefill(st):
    from pythonintern_b200 import kernels
    c = st["case"]
    return [kernels.prefill_attention_q8(st["q"], c["nq"], c["nkv"], c["hd"], st["k"], st["v"], st["ks"], st["vs"], 0,
                                         st["tables"], st["seq_start"], c["requests"], 1.0 / math.sqrt(c["hd"]),
                                         seq_ctx0=st["ctx0"])]


# --------------------------------------------------------------------------- plain forms
def _plain_tables(st):
    tables, lens, new, ring, free = st["tables"], st["lens"], st["new"], st["ring"], st["free"]
    pool, tokens = ring.numel(), st["tokens"]
    dev = tables.device
    # extend: each request takes blocks for its new tokens from the head of the ring, in order
    held = (lens + (BLOCK - 1)) // BLOCK
    want = (lens + new + (BLOCK - 1)) // BLOCK
    need = want - held
    first = torch.cumsum(need, 0) - need
    col = torch.arange(tables.shape[1], device=dev)
    take = (col >= held[:, None]) & (col < want[:, None])
    at = (free[0] + first[:, None] + col - held[:, None]) % pool
    tables.copy_(torch.where(take, ring[at], tables))
    ends = torch.cumsum(new, 0)
    seq_start = torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32)
    t = torch.arange(tokens, device=dev)
    row = torch.searchsorted(ends, t, right=True)
    pos = lens[row].to(torch.int64) + t - seq_start[row]
    slots = tables[row, pos // BLOCK].to(torch.int64) * BLOCK + pos % BLOCK
    last = torch.where(new > 0, ends - 1, torch.full_like(ends, -1)).to(torch.int64)
    maps = [seq_start, pos, row.to(torch.int32), slots, (pos + 1).to(torch.int32), last]
    total = need.sum()
    free.copy_(torch.stack([(free[0] + total) % pool, free[1] - total, free[2], free[3]]))
    lens.add_(new)
    # truncate: the blocks behind each request's kept tokens go to the tail of the ring, in order
    keep = torch.minimum(st["keep"], lens)
    held = (lens + (BLOCK - 1)) // BLOCK
    kept = (keep + (BLOCK - 1)) // BLOCK
    gone = held - kept
    first = torch.cumsum(gone, 0) - gone
    drop = (col >= kept[:, None]) & (col < held[:, None])
    at = torch.where(drop, (free[0] + free[1] + first[:, None] + col - kept[:, None]) % pool, torch.full_like(col, pool))
    spare = torch.cat([ring, ring[:1]])
    spare.scatter_(0, at.reshape(-1).to(torch.int64), tables.reshape(-1))
    ring.copy_(spare[:pool])
    tables.masked_fill_(drop, -1)
    free[1] += gone.sum()
    lens.copy_(keep)
    return maps + [tables, lens, ring, free]


def _norm_rotate(x, weight, cos, sin):
    """x [tokens, heads, hd] in 32 bits: RMS norm over each head, then the rotation of its halves."""
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    half = x.shape[-1] // 2
    turned = torch.cat([-x[..., half:], x[..., :half]], dim=-1)
    return x * cos[:, None, :] + turned * sin[:, None, :]


def _plain_qkv(st):
    c = st["case"]
    nq, nkv, hd = c["nq"], c["nkv"], c["hd"]
    x = st["qkv"].float().view(st["tokens"], nq + 2 * nkv, hd)
    cos, sin = st["cos"][st["pos"]], st["sin"][st["pos"]]
    q = _norm_rotate(x[:, :nq], st["wq"], cos, sin)
    k = _norm_rotate(x[:, nq:nq + nkv], st["wk"], cos, sin)
    blk = st["tables"][st["row"].to(torch.int64), st["pos"] // BLOCK].to(torch.int64)
    return q.reshape(st["tokens"], nq * hd).to(st["qkv"].dtype), k, x[:, nq + nkv:], blk, st["pos"] % BLOCK


def _plain_write(st):
    q, k, v, blk, off = _plain_qkv(st)
    st["k"][0, blk, off] = k.to(st["k"].dtype)
    st["v"][0, blk, off] = v.to(st["v"].dtype)
    return [q, st["k"], st["v"]]


def _to_codes(x, code):
    if code == "int8":
        return torch.round(x).clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _write_tiles(cache, scales, x, tile, off, touched, code):
    """New tokens x [tokens, kv heads, hd] into the touched tiles of one 8-bit cache; returns their values."""
    n, nkv, hd = touched.numel(), x.shape[1], x.shape[2]
    ids = touched.to(torch.int64)
    fresh = torch.zeros(n, BLOCK, nkv, hd, device=x.device)
    fresh[tile, off] = x
    written = torch.zeros(n, BLOCK, dtype=torch.bool, device=x.device)
    written[tile, off] = True
    first = torch.full((n,), BLOCK, dtype=torch.int64, device=x.device).scatter_reduce_(0, tile, off, "amin")
    fresh = fresh.permute(0, 2, 1, 3)
    scale = fresh.abs().amax((2, 3)) / TOP[code]
    scale = torch.where(scale >= TINY, scale, torch.zeros_like(scale))
    before = scales[0, ids]
    scale = torch.where(first[:, None] > 0, torch.maximum(scale, before), scale)
    some = scale > 0
    inv = torch.where(some, 1.0 / scale, torch.zeros_like(scale))
    ratio = torch.where(some, before / scale, torch.zeros_like(scale))
    old = cache[0].view(torch.uint8)[ids].view(cache.dtype).float()
    slot = torch.arange(BLOCK, device=x.device)
    history = (slot < first[:, None])[:, None, :, None]
    value = torch.where(written[:, None, :, None], fresh * inv[:, :, None, None],
                        torch.where(history, old * ratio[:, :, None, None], old))
    codes = _to_codes(value, code)
    cache[0].view(torch.uint8)[ids] = codes.view(torch.uint8)
    scales[0, ids] = scale
    return (codes.float() * scale[:, :, None, None]).permute(0, 2, 1, 3)


def _plain_write_q8(st):
    q, k, v, blk, off = _plain_qkv(st)
    begins = torch.ones_like(off)
    begins[1:] = ((blk[1:] != blk[:-1]) | (st["row"][1:] != st["row"][:-1])).to(off.dtype)
    tile = torch.cumsum(begins, 0) - 1
    code = st["case"]["code"]
    kv = [_write_tiles(st[c], st[s], x, tile, off, st["touched"], code).contiguous().to(torch.bfloat16)
          for c, s, x in (("k", "ks", k), ("v", "vs", v))]
    return [q] + kv + [st["ks"], st["vs"]]


def _values(cache, scales, tables):
    """The stored values behind block tables [rows, width]: [rows, kv heads, width * 16, hd] in 32 bits."""
    at = tables.clamp_min(0).to(torch.int64)
    x = cache[0].view(torch.uint8)[at].view(cache.dtype).float() * scales[0][at][..., None, None]
    x = x.permute(0, 2, 1, 3, 4)
    return x.reshape(x.shape[0], x.shape[1], x.shape[2] * BLOCK, x.shape[4])


def _softmax_values(s, seen, v):
    """softmax(s) v over the last axis, where `seen`; zeros where a row sees nothing."""
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(total > 0, total, torch.ones_like(total))


def _plain_decode(st):
    c = st["case"]
    n, nq, nkv, hd = c["requests"], c["nq"], c["nkv"], c["hd"]
    k, v = _values(st["k"], st["ks"], st["tables"]), _values(st["v"], st["vs"], st["tables"])
    q = st["q"].float().view(n, nkv, nq // nkv, hd)
    s = (q @ k.transpose(2, 3)) / math.sqrt(hd)
    seen = torch.arange(k.shape[2], device=q.device) < st["ctx_lens"][:, None, None, None]
    return [_softmax_values(s, seen, v).reshape(n, nq * hd).to(st["q"].dtype)]


def _plain_prefill(st):
    c = st["case"]
    n, nq, nkv, hd, most = c["requests"], c["nq"], c["nkv"], c["hd"], st["most"]
    rep = nq // nkv
    start, ctx0 = st["seq_start"].to(torch.int64), st["ctx0"].to(torch.int64)
    i = torch.arange(most, device=start.device)
    q = st["q"].float()[(start[:-1, None] + i).clamp_max(st["tokens"] - 1)].view(n, most, nkv, rep, hd)
    q = q.permute(0, 2, 3, 1, 4).reshape(n, nkv, rep * most, hd)
    k, v = _values(st["k"], st["ks"], st["tables"]), _values(st["v"], st["vs"], st["tables"])
    s = ((q @ k.transpose(2, 3)) / math.sqrt(hd)).view(n, nkv, rep, most, k.shape[2])
    seen = torch.arange(k.shape[2], device=q.device) <= (ctx0[:, None] + i)[:, None, None, :, None]
    o = _softmax_values(s.view(n, nkv, rep * most, -1),
                        seen.expand(n, 1, rep, most, k.shape[2]).reshape(n, 1, rep * most, -1), v)
    o = o.view(n, nkv, rep, most, hd).permute(0, 3, 1, 2, 4).reshape(n, most, nq * hd)
    t = torch.arange(st["tokens"], device=start.device)
    row = torch.searchsorted(start[1:], t, right=True)
    return [o[row, t - start[row]].to(st["q"].dtype)]


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    ctx, new = _lengths(case)
    n, tokens = len(ctx), sum(new)
    if case["op"] == "tables":
        taken = sum(_blocks(c + m) - _blocks(c) for c, m in zip(ctx, new))
        # lengths read and written twice; each taken block read from the ring and written to the
        # table, then the other way and cleared; the maps (8 + 4 + 8 + 4 bytes a token)
        return {"bytes": 4 * n * 6 + taken * 4 * 5 + tokens * 24 + (n + 1) * 4 + n * 8, "flops": 4 * tokens}
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["op"] == "decode_q8":
        cached = sum(ctx)
        return {"bytes": cached * 2 * nkv * hd + sum(map(_blocks, ctx)) * nkv * 8 + 2 * n * nq * hd * size,
                "flops": 4 * cached * nq * hd}
    if case["op"] == "prefill_q8":
        cached = sum(c + m for c, m in zip(ctx, new))
        pairs = sum(m * c + m * (m + 1) // 2 for c, m in zip(ctx, new))
        blocks = sum(_blocks(c + m) for c, m in zip(ctx, new))
        return {"bytes": cached * 2 * nkv * hd + blocks * nkv * 8 + 2 * tokens * nq * hd * size,
                "flops": 4 * pairs * nq * hd}
    angles = min(tokens, max(c + m for c, m in zip(ctx, new))) * 2 * hd * 4
    common = tokens * ((nq + 2 * nkv) * hd * size + nq * hd * size + 12) + angles
    flops = tokens * (nq + nkv) * hd * 8
    if case["op"] == "write":
        return {"bytes": common + tokens * 2 * nkv * hd * size, "flops": flops}
    touched = sum(_blocks(c + m) - c // BLOCK for c, m in zip(ctx, new))
    # the new codes and the scales, then the touched tiles read back as bf16 values
    tile = 2 * nkv * BLOCK * hd
    return {"bytes": common + tokens * 2 * nkv * hd + touched * nkv * 16 + touched * tile * 3,
            "flops": flops + tokens * 2 * nkv * hd * 4}


# --------------------------------------------------------------------------- the definition in 64 bits
def _exact_round(x, code):
    """The nearest 8-bit code of each value, ties to the even one, out of range to the largest."""
    if code == "int8":
        return torch.round(x).clamp(-127, 127)
    power = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -30))).clamp_min(-6.0)
    step = torch.exp2(power - 3.0)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _exact_heads(x, weight, pos, st):
    """Norm and rotation of one token's heads [heads, hd] after the other, as complex numbers."""
    hd = x.shape[-1]
    y = x / (x.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt() * weight.double()
    z = torch.complex(y[..., : hd // 2], y[..., hd // 2:])
    turn = torch.complex(st["cos"].double()[pos][:, None, : hd // 2], st["sin"].double()[pos][:, None, : hd // 2])
    z = z * turn
    return torch.cat([z.real, z.imag], dim=-1)


def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers throughout
    st = prepare(case, seed)
    ctx, new = _lengths(case)
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    rep = nq // nkv
    if case["op"] in ("decode_q8", "prefill_q8"):
        prefill = case["op"] == "prefill_q8"
        out = []
        at = 0
        for s in range(case["requests"]):
            rows = new[s] if prefill else 1
            seen = ctx[s] + new[s] if prefill else ctx[s]
            q = st["q"][at:at + rows].double().view(rows, nkv, rep, hd)
            at += rows
            if seen == 0:
                out.append(torch.zeros(rows, nq * hd, dtype=torch.float64, device="cuda"))
                continue
            ids = st["tables"][s, : _blocks(seen)].tolist()
            both = []
            for c, sc in (("k", "ks"), ("v", "vs")):
                x = torch.stack([st[c][0, b] for b in ids]) if case["code"] == "int8" else \
                    torch.stack([st[c][0, b].view(torch.int8) for b in ids]).view(torch.float8_e4m3fn)
                x = x.double() * torch.stack([st[sc][0, b] for b in ids]).double()[:, :, None, None]
                both.append(x.transpose(1, 2).reshape(-1, nkv, hd)[:seen])
            score = torch.einsum("tgrd,kgd->grtk", q, both[0]) * hd ** -0.5
            if prefill:
                i = torch.arange(rows, device="cuda")[:, None] + ctx[s]
                score = score.masked_fill(torch.arange(seen, device="cuda")[None, :] > i, -math.inf)
            o = torch.einsum("grtk,kgd->tgrd", torch.softmax(score, dim=-1), both[1])
            out.append(o.reshape(rows, nq * hd))
        return [torch.cat(out)]
    x = st["qkv"].double().view(-1, nq + 2 * nkv, hd)
    q = _exact_heads(x[:, :nq], st["wq"], st["pos"], st).reshape(-1, nq * hd)
    k = _exact_heads(x[:, nq:nq + nkv], st["wk"], st["pos"], st)
    v = x[:, nq + nkv:]
    spans = []  # (block id, first slot, first token, tokens)
    at = 0
    for s, (c, n) in enumerate(zip(ctx, new)):
        ids, p = st["tables"][s].tolist(), c
        while p < c + n:
            m = min(BLOCK - p % BLOCK, c + n - p)
            spans.append((ids[p // BLOCK], p % BLOCK, at + p - c, m))
            p += m
        at += n
    if case["op"] == "write":
        caches = []
        for name, y in (("k", k), ("v", v)):
            cache = st[name].double()
            for b, off, t, m in spans:
                cache[0, b, off:off + m] = y[t:t + m]
            caches.append(cache)
        return [q] + caches
    values, scales = [], []
    for name, sname, y in (("k", "ks", k), ("v", "vs", v)):
        scale, tiles = st[sname].double(), []
        for b, off, t, m in spans:
            fresh = y[t:t + m].transpose(0, 1)
            s = fresh.abs().amax((1, 2)) / TOP[case["code"]]
            tile = st[name][0, b].double()
            if off:
                was = scale[0, b].clone()
                s = torch.maximum(s, was)
                tile[:, :off] = _exact_round(tile[:, :off] * (was / s)[:, None, None], case["code"])
            tile[:, off:off + m] = _exact_round(fresh / s[:, None, None], case["code"])
            scale[0, b] = s
            tiles.append((tile * s[:, None, None]).transpose(0, 1))
        values.append(torch.stack(tiles))
        scales.append(scale)
    return [q] + values + scales
