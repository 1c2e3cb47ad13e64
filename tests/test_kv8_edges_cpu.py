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
