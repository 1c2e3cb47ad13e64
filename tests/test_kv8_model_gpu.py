"""The model and the engine over an 8-bit KV pool, with per-head norms, and over device block tables (GPU).

The operators have tests of their own against plain 64-bit forms; here the model's paths are compared with the
same operators called one by one, and with each other, bit for bit.
"""

import math

import numpy as np
import pytest
import torch

from pythonintern_b200 import _lib, kernels
from pythonintern_b200.config import KVCacheConfig, ModelConfig, ShardConfig

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _config(dtype="bfloat16", qk_norm=False, hd=64, **kw):
    return ModelConfig(vocab_size=128, hidden_dim=4 * hd, num_layers=2, num_heads=4, num_kv_heads=2,
                       intermediate_dim=256, max_seq_len=256, dtype=dtype, qk_norm=qk_norm, **kw)


def _fill(module, seed):
    g = torch.Generator(device="cpu").manual_seed(seed)
    with torch.no_grad():
        for name, p in sorted(module.named_parameters()):
            x = torch.randn(p.shape, generator=g)
            p.copy_((1.0 + 0.2 * x if "norm" in name else x / math.sqrt(p.shape[-1])).to(p.dtype))


def _model(cfg, seed=0):
    from pythonintern_b200.model.llama import DistributedLLaMAModel
    m = DistributedLLaMAModel(cfg, device=DEV)
    _fill(m, seed)
    return m


def _pool(cfg, kv_dtype, blocks=32):
    from pythonintern_b200.model.kv_cache import PhysicalKVCachePool
    return PhysicalKVCachePool(blocks, 16, cfg.num_kv_heads, cfg.head_dim, cfg.num_layers, device=DEV,
                               dtype=cfg.dtype, kv_dtype=kv_dtype)


@pytest.mark.parametrize("kv_dtype", ["model", "int8", "fp8_e4m3"])
@pytest.mark.parametrize("dtype,hd", [("bfloat16", 64), ("bfloat16", 128), ("float32", 32)])
def test_attention_layer_is_its_operators_in_turn(kv_dtype, dtype, hd):
    from pythonintern_b200.model.attention import DistributedAttention
    from pythonintern_b200.model.metadata import build_metadata, build_prefill_metadata
    cfg = _config(dtype, qk_norm=True, hd=hd)
    att = DistributedAttention(cfg, 1, device=DEV)
    _fill(att, 3)
    nq, nkv = 4, 2
    lens, tables = [5, 33, 16], [[3], [7, 1, 9], [4, 2]]
    a, b = _pool(cfg, kv_dtype), _pool(cfg, kv_dtype)
    g = torch.Generator(device="cpu").manual_seed(4)
    steps = [(build_prefill_metadata(lens, tables, DEV), sum(lens)),
             (build_metadata([[5], [33], [16]], tables, False, DEV, masked_padding=True), 3)]
    for md, n in steps:
        x = torch.randn(n, cfg.hidden_dim, generator=g).to(DEV, _lib.torch_dtype(dtype))
        got = att.attend(x, md, a)
        qkv = kernels.linear_qkv(x, att.q_proj.packed_weight(), att.k_proj.packed_weight(), att.v_proj.packed_weight())
        q = torch.empty(n, nq * hd, dtype=x.dtype, device=DEV)
        write = (qkv, nq, nkv, hd, att.q_norm.weight, att.k_norm.weight, cfg.rms_norm_eps, md.rope_pos, md.store_pos,
                 md.table_index, md.tables, att.rope.cos_cached, att.rope.sin_cached, q, b.k_cache, b.v_cache)
        scale = 1.0 / math.sqrt(hd)
        if kv_dtype == "model":
            kernels.qk_norm_rope_kv_write(*write, 1)
            if md.is_prefill and dtype == "bfloat16":
                want = kernels.prefill_attention(q, nq, nkv, hd, b.k_cache, b.v_cache, 1, md.tables, md.seq_start, 3, scale)
            else:
                want = kernels.paged_attention(q, nq, nkv, hd, b.k_cache, b.v_cache, 1, md.tables, md.table_index,
                                               md.ctx_lens, False, scale,
                                               num_splits=kernels.attention_splits(n, nkv, md.max_ctx, 16, DEV))
        else:
            kernels.qk_norm_rope_kv_write_q8(*write, b.k_scale, b.v_scale, 1)
            cache = (q, nq, nkv, hd, b.k_cache, b.v_cache, b.k_scale, b.v_scale, 1, md.tables)
            if md.is_prefill:
                want = kernels.prefill_attention_q8(*cache, md.seq_start, 3, scale)
            else:
                want = kernels.paged_attention_q8(*cache, md.table_index, md.ctx_lens, False, scale)
        _lib.check_device_status(DEV, "layer")
        assert torch.equal(got, want) and torch.isfinite(got.float()).all()
        assert torch.equal(a.k_cache.view(torch.uint8), b.k_cache.view(torch.uint8))
    k, v = a.read_kv_sequence(1, tables[1], 34)
    assert k.shape == v.shape == (34, nkv, hd) and k.dtype == a.dtype and (k != 0).any() and (v != 0).any()
    assert a.read_kv_sequence(1, [], 0)[0].shape == (0, nkv, hd)


@pytest.mark.parametrize("kv_dtype", ["int8", "fp8_e4m3"])
@pytest.mark.parametrize("masked", [True, False])
def test_engine_over_an_8_bit_pool(kv_dtype, masked):
    """Prompts of several lengths, then decode steps: graphs and eager steps agree bit for bit, and the values
    read back differ from a pool of the model's type by no more than their rounding in the first layer."""
    from pythonintern_b200.worker.execution_engine import WorkerExecutionEngine
    from pythonintern_b200.worker.messages import SequenceSlot, StepRequest

    def run(kind, graphs):
        cfg = _config(masked_decode_padding=masked)
        eng = WorkerExecutionEngine(cfg, ShardConfig(), KVCacheConfig(16, 32, DEV, kv_dtype=kind), None, DEV,
                                    use_cuda_graphs=graphs)
        _fill(eng.model, 8)
        rng = np.random.default_rng(5)
        prompts = [rng.integers(0, 128, n).tolist() for n in (1, 15, 16, 40)]
        tables = [eng.kv_manager.allocate_blocks_for_sequence(str(i), len(p) + 6) for i, p in enumerate(prompts)]
        rows, out = [t.physical_block_ids for t in tables], []
        r = eng.execute_step(StepRequest(step_id=0, active_sequences=[
            SequenceSlot(seq_id=str(i), is_prefill=True, prompt_token_ids=p, block_table=rows[i])
            for i, p in enumerate(prompts)]))
        cur = [t.token_id for t in r.sampled_tokens]
        out.append([t.top_logits for t in r.sampled_tokens])
        first = [eng.kv_manager.pool.read_kv_sequence(0, rows[i], len(p)) for i, p in enumerate(prompts)]
        for step in range(4):
            r = eng.execute_step(StepRequest(step_id=1 + step, active_sequences=[
                SequenceSlot(seq_id=str(i), is_prefill=False, current_token_id=cur[i],
                             current_len=len(p) + step + 1, block_table=rows[i]) for i, p in enumerate(prompts)]))
            cur = [t.token_id for t in r.sampled_tokens]
            out.append([t.top_logits for t in r.sampled_tokens])
        return out, first

    eager, first = run(kv_dtype, False)
    graph, _ = run(kv_dtype, True)
    assert eager == graph
    assert np.isfinite(np.asarray(eager)).all()
    _, exact = run("model", False)
    # Layer 0's K and V come from the same bf16 inputs.  The exact pool rounds them to bf16 (2^-8 of the value) after
    # the rotation; the 8-bit one rounds the value before that rounding (int8: half a step of amax / 127; e4m3: 2^-4
    # of the value or half a step of 2^-9 below 2^-6, in units of amax / 448), and the read rounds to bf16 again.
    for (k8, v8), (k, v) in zip(first, exact):
        for got, want in ((k8, k), (v8, v)):
            amax = want.double().abs().max() * (1 + 2.0 ** -8)
            code = amax / 254 if kv_dtype == "int8" else want.double().abs() * 2.0 ** -4 * (1 + 2.0 ** -8) + amax / 448 * 2.0 ** -10
            tol = code * (1 + 2.0 ** -8) + want.double().abs() * 2 * 2.0 ** -8 * (1 + 2.0 ** -6)
            assert ((got.double() - want.double()).abs() <= tol).all()


@pytest.mark.parametrize("kv_dtype", ["model", "int8"])
def test_device_block_tables_drive_the_model(kv_dtype):
    """Prompts, drafts of five tokens, a truncation and another step: the same tokens and pool as with host tables."""
    from pythonintern_b200.model.kv_cache import DeviceBlockTables, KVCacheManager
    from pythonintern_b200.model.metadata import build_prefill_metadata
    cfg = _config(qk_norm=True)
    model = _model(cfg, 2)
    bt = DeviceBlockTables(3, 8, 32, device=DEV)
    host = KVCacheManager(KVCacheConfig(16, 32, DEV, kv_dtype=kv_dtype), cfg, 1)
    pools = host.pool, _pool(cfg, kv_dtype)
    g = torch.Generator(device="cpu").manual_seed(1)
    have = [0, 0, 0]
    for step, (new, keep) in enumerate([([7, 30, 16], None), ([5, 5, 5], [9, 31, 16]), ([5, 3, 1], None)]):
        ids = torch.randint(0, 128, (1, sum(new)), generator=g).to(DEV)
        tables = []
        for s in range(3):
            tables.append(list(host.allocate_blocks_for_sequence(str(s), have[s] + new[s]).physical_block_ids))
        want_md = build_prefill_metadata(new, tables, DEV, ctx0=have)
        md = bt.extend(new) if step != 1 else bt.extend(torch.tensor(new, dtype=torch.int32, device=DEV), sum(new))
        for name in ("rope_pos", "table_index", "ctx_lens", "seq_start", "seq_ctx0", "last_rows"):
            assert torch.equal(getattr(md, name), getattr(want_md, name)), name
        want, want_top = model.greedy(ids, None, pools[0], tables, True, step, metadata=want_md)
        got, top = model.greedy(ids, None, pools[1], tables, True, step, metadata=md)
        _lib.check_device_status(DEV, "step")
        assert torch.equal(got, want) and torch.equal(top, want_top)
        have = [h + n for h, n in zip(have, new)]
        if keep is not None:
            bt.truncate(keep)
            have = keep
            for s in range(3):  # the host's blocks behind the kept tokens
                t = host.block_tables[str(s)]
                kept = -(-keep[s] // 16)
                host.free_blocks.extend(t.physical_block_ids[kept:])
                del t.physical_block_ids[kept:]
        assert bt.lens.tolist() == have
    assert torch.equal(pools[0].k_cache.view(torch.uint8), pools[1].k_cache.view(torch.uint8))
    assert torch.equal(pools[0].v_cache.view(torch.uint8), pools[1].v_cache.view(torch.uint8))
    bt.truncate([0, 0, 0])
    assert bt.free_state[:2].tolist()[1] == 32 and (bt.tables == -1).all()


def test_a_step_that_cannot_be_served_is_empty():
    from pythonintern_b200.model.kv_cache import DeviceBlockTables
    cfg = _config()
    model, pool = _model(cfg), _pool(cfg, "int8")
    bt = DeviceBlockTables(2, 8, 3, device=DEV)
    bt.extend([16, 20])
    before = pool.k_cache.clone(), bt.tables.clone(), bt.lens.clone()
    md = bt.extend([1, 0])
    model.forward_hidden(torch.zeros(1, 1, dtype=torch.int64, device=DEV), md, pool)
    with pytest.raises((MemoryError, IndexError)):
        _lib.check_device_status(DEV, "step")
    _lib.check_device_status(DEV, "cleared")
    assert torch.equal(pool.k_cache, before[0]) and torch.equal(bt.tables, before[1]) and torch.equal(bt.lens, before[2])


@pytest.mark.parametrize("kv_dtype", ["model", "fp8_e4m3"])
def test_idle_slots_and_captured_steps_over_device_tables(kv_dtype):
    """Slots without new tokens, and a step of drafts (extend, forward, truncate) captured once and replayed with
    other lengths on the device: the same as eager steps over a second set of tables and pool."""
    from pythonintern_b200.model.kv_cache import DeviceBlockTables
    cfg = _config()
    model = _model(cfg, 6)
    sides = [(DeviceBlockTables(4, 8, 32, device=DEV), _pool(cfg, kv_dtype)) for _ in range(2)]
    g = torch.Generator(device="cpu").manual_seed(3)
    prompt = torch.randint(0, 128, (1, 41), generator=g).to(DEV)
    for bt, pool in sides:
        model.greedy(prompt, None, pool, [], True, 0, metadata=bt.extend([30, 0, 11, 0]))
    _lib.check_device_status(DEV, "prompts")
    new = torch.zeros(4, dtype=torch.int32, device=DEV)
    keep = torch.zeros(4, dtype=torch.int32, device=DEV)
    ids = torch.zeros(1, 8, dtype=torch.int64, device=DEV)

    def step(bt, pool):
        out = model.greedy(ids, None, pool, [], True, 0, metadata=bt.extend(new, 8))
        bt.truncate(keep)
        return out

    plan = [([5, 0, 3, 0], [33, 0, 14, 0]), ([2, 5, 0, 1], [35, 2, 14, 1]), ([0, 4, 2, 2], [17, 6, 16, 0])]
    (bt, pool), (bt2, pool2) = sides
    want = []
    for k, (n, c) in enumerate(plan):
        ids.copy_(torch.randint(0, 128, (1, 8), generator=torch.Generator().manual_seed(k)))
        new.copy_(torch.tensor(n, dtype=torch.int32))
        keep.copy_(torch.tensor(c, dtype=torch.int32))
        tok, top = step(bt, pool)
        active = torch.tensor(n) > 0
        want.append((tok.cpu()[active], top.cpu()[active], bt.tables.clone(), bt.lens.clone(), bt.free_state.clone()))
    _lib.check_device_status(DEV, "eager")
    new.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tok, top = step(bt2, pool2)
    for k, (n, c) in enumerate(plan):
        ids.copy_(torch.randint(0, 128, (1, 8), generator=torch.Generator().manual_seed(k)))
        new.copy_(torch.tensor(n, dtype=torch.int32))
        keep.copy_(torch.tensor(c, dtype=torch.int32))
        graph.replay()
        active = torch.tensor(n) > 0
        got = (tok.cpu()[active], top.cpu()[active], bt2.tables, bt2.lens, bt2.free_state)
        assert all(torch.equal(a, b) for a, b in zip(got, want[k])), k
    _lib.check_device_status(DEV, "replays")
    assert torch.equal(pool.k_cache.view(torch.uint8), pool2.k_cache.view(torch.uint8))


def test_qk_norm_adds_two_keys_to_a_layer_and_none_without():
    plain, normed = _model(_config()).state_dict(), _model(_config(qk_norm=True)).state_dict()
    extra = set(normed) - set(plain)
    assert set(plain) <= set(normed)
    assert extra == {f"layers.{i}.self_attn.{n}_norm.weight" for i in range(2) for n in "qk"}
