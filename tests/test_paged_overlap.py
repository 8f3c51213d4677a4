"""What a paged call writes may not lie in what its blocks read (no GPU needed: ranges are compared before any
pointer is looked at)."""
import ctypes as C

import pytest

from sharpinference_b200 import native

N = native
AT = dict(pages=1 << 32, page_table=2 << 32, row_starts=3 << 32, lengths=4 << 32, qkv=5 << 32, query=6 << 32,
          frequencies=7 << 32, output=8 << 32, workspace=9 << 32, keys=10 << 32, values=11 << 32)
STREAMS, WIDTH, ROWS, HEADS = 2, 4, 5, 4
# 8 pages of 64 tokens, 2 heads of 128; rows of 512 query values and 1024 in all
SIZE = dict(pages=8 * 64 * 2 * 128 * 2 * 9 // 16, page_table=4 * STREAMS * WIDTH, row_starts=4 * (STREAMS + 1),
            lengths=4 * STREAMS, qkv=ROWS * 1024 * 4, query=ROWS * 512 * 4, frequencies=48 * 4, output=ROWS * 512 * 4,
            keys=ROWS * 256 * 4, values=ROWS * 256 * 4)


def _cache(at):
    return native.PagedCache(pages=at["pages"], page_table=at["page_table"], page_count=8, streams=STREAMS,
                             table_width=WIDTH, page_size=64, kv_heads=2, head_size=128)


def _append(at):
    return N.lib.si_paged_rope_kv_append(C.byref(_cache(at)), N.F32, at["qkv"], 1024, at["row_starts"], at["lengths"],
                                         at["frequencies"], at["query"], 512, ROWS, HEADS, 96, 1.0, None)


def _gather(at):
    return N.lib.si_paged_kv_gather(C.byref(_cache(at)), N.F32, at["row_starts"], at["lengths"], at["keys"],
                                    at["values"], ROWS, None)


def _attend(at):
    return N.lib.si_paged_attention(C.byref(_cache(at)), N.F32, at["query"], 512, at["row_starts"], at["lengths"],
                                    at["output"], 512, ROWS, ROWS, HEADS, 0.1, 0, at["workspace"], 1 << 31, None)


READ = ["page_table", "row_starts", "lengths"]
CASES = [(_append, w, r) for w, r in [("query", "pages"), ("query", "frequencies"), ("pages", "qkv")]]
CASES += [(_append, "query", r) for r in READ] + [(_gather, w, r) for w in ("keys", "values") for r in ["pages"] + READ]
CASES += [(_attend, w, r) for w in ("output", "workspace") for r in ["pages"] + READ] + [(_attend, "workspace", "query")]


@pytest.mark.parametrize("call,written,read", CASES)
def test_overlaps_are_refused(call, written, read):
    for where in (AT[read], AT[read] + SIZE[read] - 4):
        at = dict(AT, **{written: where // 16 * 16})
        assert call(at) == N.SI_ERR_INVALID_ARGUMENT
        assert N.last_error() == f"port '{written}': overlaps port '{read}'"
    for where in (AT[read] + (SIZE[read] + 15) // 16 * 16,):  # next to it
        assert call(dict(AT, **{written: where})) == N.SI_ERR_INVALID_ARGUMENT  # no device memory here
        assert "overlaps" not in N.last_error()


@pytest.mark.parametrize("call", [_append, _gather, _attend])
def test_tensors_apart_are_not_refused_as_overlapping(call):
    assert call(AT) == N.SI_ERR_INVALID_ARGUMENT
    assert "overlaps" not in N.last_error()
