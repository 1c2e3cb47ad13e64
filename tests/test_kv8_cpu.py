"""Refusals of the 8-bit KV cache entry points that need no GPU: the C ABI's argument checks."""

import pytest

from pythonintern_b200 import _lib

A = 1 << 20  # an aligned address that no rejected call dereferences


def refused(rc, code, text):
    assert rc == code, (rc, _lib.last_error())
    assert text in _lib.last_error()


def _write(q8=False, n=1, nq=4, nkv=2, hd=64, ld=None, rows=1, blocks=4, bs=16, qkv=A, layer=0, dtype=1, cache=2,
           scale=A):
    L = _lib.lib()
    ld = (nq + 2 * nkv) * hd if ld is None else ld
    args = [qkv, ld, n, nq, nkv, hd, None, None, 1e-5, A, None, None, A, rows, 1, blocks, bs, A, A, 64, A, A, A]
    if q8:
        return L.b2_qk_norm_rope_kv_write_q8(*args, scale, scale, cache, layer, dtype, None, None)
    return L.b2_qk_norm_rope_kv_write(*args, layer, dtype, None, None)


def test_write_refusals():
    for q8 in (False, True):
        refused(_write(q8, nq=0), _lib.B2_EINVAL, "head counts")
        refused(_write(q8, dtype=7), _lib.B2_EINVAL, "dtype")
        refused(_write(q8, hd=96), _lib.B2_ENOTSUP, "head_dim 96")
        refused(_write(q8, ld=10), _lib.B2_EINVAL, "ld_qkv")
        refused(_write(q8, blocks=0), _lib.B2_EINVAL, "geometry")
        refused(_write(q8, layer=-1), _lib.B2_EINVAL, "geometry")
        refused(_write(q8, qkv=None), _lib.B2_EINVAL, "null")
        refused(_write(q8, qkv=A + 4), _lib.B2_EINVAL, "aligned")
        refused(_write(q8, n=2), _lib.B2_EINVAL, "table rows")
        assert _write(q8, n=0) == _lib.B2_OK
    refused(_write(True, bs=32), _lib.B2_ENOTSUP, "block_size 32")
    refused(_write(True, cache=1), _lib.B2_EINVAL, "cache dtype")
    refused(_write(True, scale=None), _lib.B2_EINVAL, "null scales")


def _attend(prefill=False, n=1, nq=4, nkv=2, hd=64, ld=None, rows=1, blocks=4, bs=16, q=A, layer=0, dtype=1, cache=2,
            stride=1, lens=A):
    L = _lib.lib()
    ld = nq * hd if ld is None else ld
    head = [q, ld, n, nq, nkv, hd, A, A, A, A, cache, layer, blocks, bs, A, rows, stride]
    tail = [1.0, A, nq * hd, dtype, A, 1 << 40, None, None]
    if prefill:
        return L.b2_prefill_attention_q8(*head, lens, None, 1, *tail)
    return L.b2_paged_attention_q8(*head, None, lens, 0, *tail)


def test_attention_refusals():
    for pre in (False, True):
        refused(_attend(pre, nq=3), _lib.B2_EINVAL, "head counts")
        refused(_attend(pre, dtype=2), _lib.B2_EINVAL, "dtype")
        refused(_attend(pre, cache=0), _lib.B2_EINVAL, "cache dtype")
        refused(_attend(pre, hd=96), _lib.B2_ENOTSUP, "head_dim 96")
        refused(_attend(pre, nq=34), _lib.B2_ENOTSUP, "nq/nkv = 17")
        refused(_attend(pre, bs=8), _lib.B2_ENOTSUP, "block_size 8")
        refused(_attend(pre, ld=8), _lib.B2_EINVAL, "strides")
        refused(_attend(pre, blocks=0), _lib.B2_EINVAL, "geometry")
        refused(_attend(pre, stride=1 << 28), _lib.B2_EINVAL, "too large")
        refused(_attend(pre, q=None), _lib.B2_EINVAL, "null")
        refused(_attend(pre, q=A + 2), _lib.B2_EINVAL, "aligned")
        refused(_attend(pre, lens=None), _lib.B2_EINVAL, "null")
        assert _attend(pre, n=0) == _lib.B2_OK
    refused(_attend(False, n=2), _lib.B2_EINVAL, "table rows")
    refused(_attend(True, rows=0), _lib.B2_EINVAL, "geometry")


def test_read_refusals():
    def read(cache=3, out=1, hd=64, n=1, ids=A, k=A, bs=16):
        return _lib.lib().b2_kv_read_q8(k, A, A, A, cache, 0, 4, bs, 2, hd, ids, n, A, A, out, None, None)
    refused(read(cache=1), _lib.B2_EINVAL, "cache dtype")
    refused(read(out=3), _lib.B2_EINVAL, "dtype")
    refused(read(hd=80), _lib.B2_ENOTSUP, "head_dim 80")
    refused(read(n=-1), _lib.B2_EINVAL, "geometry")
    refused(read(ids=None), _lib.B2_EINVAL, "null")
    refused(read(k=A + 8), _lib.B2_EINVAL, "aligned")
    refused(read(bs=4), _lib.B2_ENOTSUP, "block_size 4")
    assert read(n=0) == _lib.B2_OK


def test_block_tables_refusals():
    L = _lib.lib()

    def extend(n=2, stride=4, bs=16, ring=A, state=A, blocks=8, most=4, lens=A, maps=A):
        return L.b2_block_tables_extend(A, n, stride, lens, A, bs, ring, blocks, state, most, A, maps, maps, maps,
                                        maps, A, None, None)
    refused(extend(n=0), _lib.B2_EINVAL, "sizes")
    refused(extend(bs=0), _lib.B2_EINVAL, "sizes")
    refused(extend(most=-1), _lib.B2_EINVAL, "sizes")
    refused(extend(n=16385), _lib.B2_ENOTSUP, "16384")
    refused(extend(lens=None), _lib.B2_EINVAL, "null")
    refused(extend(maps=None), _lib.B2_EINVAL, "null map")
    refused(extend(state=None), _lib.B2_EINVAL, "together")
    rc = L.b2_block_tables_truncate(A, 2, 4, A, A, 16, None, 8, A, None, None)
    refused(rc, _lib.B2_EINVAL, "null")


def test_pool_types_and_refusals():
    import torch
    from pythonintern_b200._lib import B2Error
    from pythonintern_b200.config import KVCacheConfig, ModelConfig
    from pythonintern_b200.model.kv_cache import KVCacheManager, PhysicalKVCachePool
    assert KVCacheConfig().kv_dtype == "model" and ModelConfig().qk_norm is False
    m = KVCacheManager(KVCacheConfig(16, 4, "meta", kv_dtype="int8"), ModelConfig(dtype="bfloat16"), 1)
    p = m.pool
    assert p.k_cache.shape == (8, 4, 4, 16, 64) and p.k_cache.dtype is torch.int8 and p.dtype is torch.bfloat16
    assert p.k_scale.shape == (8, 4, 4) and p.k_scale.dtype is torch.float32
    assert KVCacheManager(KVCacheConfig(16, 4, "meta", kv_dtype="fp8_e4m3"), ModelConfig(),
                          1).pool.v_cache.dtype is torch.float8_e4m3fn
    assert not KVCacheManager(KVCacheConfig(16, 4, "meta"), ModelConfig(), 1).pool.quantised
    with pytest.raises(ValueError, match="kernels only"):
        p.store_kv(0, 0, 0, torch.zeros(4, 64), torch.zeros(4, 64))
    with pytest.raises(ValueError, match="kernels only"):
        p.store_kv_batch(0, [0], [0], torch.zeros(1, 4, 64), torch.zeros(1, 4, 64))
    for bs, hd in ((8, 64), (16, 96)):
        with pytest.raises(ValueError, match="blocks of 16"):
            PhysicalKVCachePool(4, bs, 4, hd, 1, device="meta", dtype="bfloat16", kv_dtype="int8")
    with pytest.raises(B2Error, match="unsupported KV cache dtype"):
        PhysicalKVCachePool(4, 16, 4, 64, 1, device="meta", kv_dtype="int4")


def test_device_block_tables_refusals():
    import torch
    from pythonintern_b200.model.kv_cache import DeviceBlockTables
    bt = DeviceBlockTables(3, 4, 8, device="cpu")
    with pytest.raises(ValueError, match="n_tokens"):
        bt.extend(torch.ones(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="at least one"):
        bt.extend([0, 0, 0])
    for bad in ([1, 2], torch.ones(3, dtype=torch.int64), torch.ones(2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="per sequence slot"):
            bt.truncate(bad)


def test_norms_of_q_and_k_are_the_same_on_every_rank():
    import torch
    from pythonintern_b200.config import ModelConfig
    from pythonintern_b200.tensor_parallel.sharding import WeightSharder
    state = {"layers.0.self_attn.q_norm.weight": torch.arange(8.0), "layers.0.self_attn.k_norm.weight": torch.ones(8),
             "layers.0.self_attn.q_proj.weight": torch.zeros(16, 32)}
    for rank in range(2):
        shard = WeightSharder(ModelConfig(hidden_dim=32, num_heads=4, num_kv_heads=2), 2).shard_full_model_state_dict(state, rank)
        for n in "qk":
            key = f"layers.0.self_attn.{n}_norm.weight"
            assert torch.equal(shard[key], state[key])
        assert shard["layers.0.self_attn.q_proj.weight"].shape == (16, 16)
