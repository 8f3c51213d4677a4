"""Paged calls of many rows and many streams: blocks that take several rows together, and searches among more streams
than a warp has lanes."""
import ctypes as C

import numpy as np
import pytest

import paged_reference as ref
from sharpinference_b200 import native
from test_paged_gpu import TYPES, Device, check_attention, gather

pytestmark = pytest.mark.gpu
N = native


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


# a block takes 2, 4, 8 rows from 16, 32, 64 rows an SM on; 148 SMs
MANY = [[2368, 0, 1, 90], [2000, 700, 2100], [4740, 33], [9472, 5], [1] * 7 + [9600, 0, 300]]


@pytest.mark.parametrize("type", [N.F32, N.F16])
@pytest.mark.parametrize("rows", MANY)
@pytest.mark.parametrize("d,kv", [(64, 1), (128, 3)])
def test_gather_of_many_rows_is_exact(torch, type, rows, d, kv):
    s = ref.Streams(np.random.default_rng(d), [n + 21 * b for b, n in enumerate(rows)], kv, d, 64)
    s.unmap(0, 1)
    k, v = gather(torch, Device(torch, s), rows, type)
    for got, have in ((k, s.keys), (v, s.values)):
        want = []
        for b, n in enumerate(rows):
            t = np.arange(s.lengths[b] - n, s.lengths[b])
            want.append(have[b][t] * s.mapped[b][t // 64][:, None, None])
        assert np.array_equal(got, np.concatenate(want).reshape(got.shape))


@pytest.mark.parametrize("type", [N.F32, N.F16])
@pytest.mark.parametrize("rows", MANY)
@pytest.mark.parametrize("d,kv,heads,rotary,pad", [(64, 1, 1, 64, 0), (128, 2, 4, 96, 8), (192, 1, 3, 10, 3),
                                                   (128, 1, 2, 0, 0)])
def test_append_of_many_rows_stores_what_single_rows_store(torch, type, rows, d, kv, heads, rotary, pad):
    """One call against calls of 500 rows at most, which take a row to a block: the same bytes and queries."""
    lengths = [n + 21 * b for b, n in enumerate(rows)]
    s = ref.Streams(np.random.default_rng(d), lengths, kv, d, 64)
    dev, total, width, q = Device(torch, s), sum(rows), (heads + 2 * kv) * d, heads * d
    dt = torch.float32 if type == N.F32 else torch.float16
    x = torch.randn(total, width + pad, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(dt)
    freq = torch.from_numpy((10000.0 ** (-np.arange(0, max(rotary, 2), 2) / max(rotary, 2))).astype(np.float32)).cuda()
    clean = dev.pool.clone()

    def append(first, starts, lengths):
        n = starts[-1]
        out = torch.full((n, q + pad), 9.0, dtype=dt, device="cuda")
        st, ln = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (starts, lengths))
        torch.cuda.synchronize()
        native.call("si_paged_rope_kv_append", C.byref(dev.cache), type, x[first:].data_ptr(), width + pad,
                    st.data_ptr(), ln.data_ptr(), freq.data_ptr(), out.data_ptr(), q + pad, n, heads, rotary, 1.19, None)
        torch.cuda.synchronize()
        return out

    got = append(0, [0] + np.cumsum(rows).tolist(), lengths)
    pool = dev.pool.clone()
    dev.pool.copy_(clean)
    first = 0
    for b, n in enumerate(rows):
        for i in range(0, n, 500):
            m = min(500, n - i)
            starts = [0] * (b + 1) + [m] * (len(rows) - b)
            want = append(first, starts, [lengths[b] - n + i + m] * len(rows))
            assert torch.equal(got[first:first + m], want)
            first += m
    assert torch.equal(pool, dev.pool)
    assert not torch.equal(pool, clean)


@pytest.mark.parametrize("type", [N.F32, N.F16])
@pytest.mark.parametrize("streams", [32, 33, 64, 65, 150, 700])
@pytest.mark.parametrize("rows", [[1], [1, 0, 3], [0, 0, 5, 1]])
def test_few_rows_of_many_streams(torch, type, streams, rows):
    rng = np.random.default_rng(streams)
    rows = [rows[b % len(rows)] for b in range(streams)]
    lengths = [n + int(x) for n, x in zip(rows, 200 * rng.random(streams) ** 4)]
    s = ref.Streams(rng, lengths, 2, 64, 16)
    check_attention(torch, s, rows, 4, type=type)


@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("streams", [33, 40, 96, 130])
@pytest.mark.parametrize("rows", [[40, 1, 0], [0, 0, 0, 33, 150], [0] * 37 + [36]])
def test_chunks_of_many_streams(torch, streams, rows, window):
    rng = np.random.default_rng(streams)
    rows = [rows[b % len(rows)] for b in range(streams)]
    if not sum(rows):
        rows[-1] = 36
    lengths = [n + int(x) for n, x in zip(rows, 150 * rng.random(streams) ** 3)]
    s = ref.Streams(rng, lengths, 1, 64, 16)
    check_attention(torch, s, rows, 1, window=window)
    check_attention(torch, s, rows, 1, window=window, type=N.F16)


def test_one_long_stream_among_many(torch):
    """The cut's search meets a stream that is most of the line."""
    rng = np.random.default_rng(9)
    lengths = [3] * 45 + [9000] + [17] * 40
    s = ref.Streams(rng, lengths, 1, 128, 64)
    for type in TYPES:
        check_attention(torch, s, [1] * 86, 2, type=type)
