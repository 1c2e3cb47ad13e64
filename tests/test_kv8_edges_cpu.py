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
