"""Refusals around the 8-bit KV cache that need no GPU."""

import pytest

from pythonintern_b200 import _lib
from test_kv8_cpu import A, refused


@pytest.mark.parametrize("fn", ["b2_block_tables_extend", "b2_block_tables_extend_filled"])
def test_both_forms_of_extend_refuse_the_same(fn):
    def extend(n=2, stride=4, bs=16, ring=A, state=A, most=4, lens=A, maps=A):
        return getattr(_lib.lib(), fn)(A, n, stride, lens, A, bs, ring, 8, state, most, A, maps, maps, maps, maps, A,
                                       None, None)
    for kw, code, text in ((dict(n=0), _lib.B2_EINVAL, "sizes"), (dict(bs=0), _lib.B2_EINVAL, "sizes"),
                           (dict(most=-1), _lib.B2_EINVAL, "sizes"), (dict(n=16385), _lib.B2_ENOTSUP, "16384"),
                           (dict(lens=None), _lib.B2_EINVAL, "null"), (dict(maps=None), _lib.B2_EINVAL, "null map"),
                           (dict(state=None), _lib.B2_EINVAL, "together")):
        refused(extend(**kw), code, text)
        assert _lib.last_error().startswith(fn + ":")


@pytest.mark.parametrize("source", ["attention_q8.cu", "prefill_q8_tc.cu", "qk_norm_rope.cu", "block_tables.cu", "q8.cuh"])
def test_kernels_that_begin_early_do_not_load_through_the_read_only_path(source):
    """Tables, scales and codes may be written by the kernel before, which need not have ended when these begin:
    ld.global.nc wants memory that nobody writes for as long as the kernel lives."""
    import os
    text = open(os.path.join(os.path.dirname(_lib.LIB_PATH), "csrc", source)).read()
    for word in ("__ldg", "global.nc", "__restrict__"):
        assert word not in text, word


@pytest.mark.parametrize("kv_dtype", ["int8", "fp8_e4m3"])
def test_a_pool_that_no_kernel_reads_is_refused_with_its_model(kv_dtype):
    from pythonintern_b200.config import KVCacheConfig, ModelConfig
    from pythonintern_b200.model.kv_cache import KVCacheManager

    def manager(heads, kv_heads, kind):
        cfg = ModelConfig(hidden_dim=32 * heads, num_heads=heads, num_kv_heads=kv_heads, dtype="bfloat16")
        return KVCacheManager(KVCacheConfig(16, 4, "meta", kv_dtype=kind), cfg, 1)

    with pytest.raises(ValueError, match="16 q heads"):
        manager(17, 1, kv_dtype)
    assert manager(32, 2, kv_dtype).pool.quantised  # 16 to 1
    assert not manager(17, 1, "model").pool.quantised


def test_norms_of_heads_that_no_kernel_serves_are_refused_with_the_layer():
    from pythonintern_b200.config import ModelConfig
    from pythonintern_b200.model.attention import DistributedAttention

    def layer(hd, qk_norm):
        return DistributedAttention(ModelConfig(hidden_dim=4 * hd, num_heads=4, num_kv_heads=2, dtype="bfloat16",
                                                max_seq_len=32, qk_norm=qk_norm), 0, device="cpu")

    for hd in (16, 96):
        with pytest.raises(ValueError, match="qk_norm"):
            layer(hd, True)
        assert layer(hd, False).q_norm is None
    assert layer(64, True).q_norm.weight.shape == (64,)
