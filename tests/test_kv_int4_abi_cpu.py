"""The C entries of the 4-bit cache: sizes that the workspace query refuses."""
import ctypes

import pytest

import int4_int8_ext as ext
from tests.test_kv_int4_cpu import _c_cache


@pytest.mark.parametrize("change", [dict(rows=-1), dict(batch=-1), dict(page_size=0), dict(page_size=-4), dict(table_cols=-1),
                                    dict(pages=-1), dict(heads=-2)], ids=str)
@pytest.mark.parametrize("max_q", [1, 200])
def test_the_workspace_query_refuses_sizes_that_the_call_refuses(change, max_q):
    import build_native

    build_native.build()
    lib, c, n = ext.lib(), _c_cache(**change), ctypes.c_size_t(7)
    assert lib.w4a8_attention_int4_workspace(ctypes.byref(c), 2, 2, max_q, 1 << 20, 0, ctypes.byref(n)) == ext.ERR_ARG
    assert n.value == 0
