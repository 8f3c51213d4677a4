"""Sizes of the paged attention's workspace are asked before a cache has its memory (no GPU needed)."""
import ctypes as C

import pytest

from sharpinference_b200 import native

N = native


def _cache(**kw):
    f = dict(page_count=8, streams=2, table_width=4, page_size=64, kv_heads=2, head_size=128)
    f.update(kw)
    return native.PagedCache(**f)


@pytest.mark.parametrize("rows,most", [(2, 1), (5, 4), (700, 512), (1, 1)])
def test_workspace_of_a_cache_without_memory(rows, most):
    bare = native.paged_attention_workspace_bytes(_cache(), rows, most, 8)
    assert bare > 0
    assert bare == native.paged_attention_workspace_bytes(_cache(pages=1 << 32, page_table=1 << 33), rows, most, 8)


def test_calls_without_row_starts_still_want_one_row_per_stream():
    cache = _cache(pages=1 << 32, page_table=2 << 32)
    assert N.lib.si_paged_kv_gather(C.byref(cache), N.F32, None, 3 << 32, 4 << 32, 5 << 32, 3,
                                    None) == N.SI_ERR_ADAPTATION
    assert "row_starts" in N.last_error()
