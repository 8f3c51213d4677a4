"""Append and attention one behind the other without a host between them: a chunk reads what the append before it
wrote, in tiles that the steps before had filled in part and read."""
import ctypes as C

import numpy as np
import pytest

import paged_reference as ref
from sharpinference_b200 import native
from test_paged_gpu import Device, gather

pytestmark = pytest.mark.gpu
N = native


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


@pytest.mark.parametrize("type", [N.F32, N.F16])
@pytest.mark.parametrize("rows,past,steps", [((37, 41), (5, 0), 6), ((21, 50), (700, 3), 5), ((150, 1), (90, 2000), 3),
                                             ((1, 1), (40, 300), 8)])
def test_chunks_read_what_the_append_before_them_wrote(torch, type, rows, past, steps):
    d, kv, heads, ps = 128, 2, 4, 32
    t, total = torch, sum(rows)
    dt = t.float32 if type == N.F32 else t.float16
    final = [p + steps * r for p, r in zip(past, rows)]
    s = ref.Streams(np.random.default_rng(total), final, kv, d, ps)
    dev = Device(torch, s)
    lengths = [t.tensor([p + (i + 1) * r for p, r in zip(past, rows)], dtype=t.int32, device="cuda")
               for i in range(steps)]
    starts = t.tensor([0, rows[0], total], dtype=t.int32, device="cuda")
    freq = (10000.0 ** (-t.arange(0, 96, 2, device="cuda") / 96)).float()
    qkv, query, out = (t.zeros(steps, total, n * d, dtype=dt, device="cuda") for n in (heads + 2 * kv, heads, heads))
    ws = t.zeros(native.paged_attention_workspace_bytes(dev.cache, total, max(rows), heads), dtype=t.uint8, device="cuda")
    t.cuda.synchronize()
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        st = t.cuda.current_stream().cuda_stream
        for i in range(steps):
            native.call("si_paged_rope_kv_append", C.byref(dev.cache), type, qkv[i].data_ptr(), qkv.shape[2],
                        starts.data_ptr(), lengths[i].data_ptr(), freq.data_ptr(), query[i].data_ptr(), heads * d, total,
                        heads, 96, 1.0, st)
            native.call("si_paged_attention", C.byref(dev.cache), type, query[i].data_ptr(), heads * d,
                        starts.data_ptr(), lengths[i].data_ptr(), out[i].data_ptr(), heads * d, total, max(rows), heads,
                        d ** -0.5, 0, ws.data_ptr(), ws.numel(), st)
    rng = np.random.default_rng(1)
    for _ in range(3):  # every replay writes other tokens over the last one's
        qkv.copy_(t.from_numpy(rng.standard_normal(tuple(qkv.shape)).astype(np.float32)))
        graph.replay()
        t.cuda.synchronize()
        assert native.device_error_take(0) == 0
        k, v = gather(torch, dev, final)
        at = np.concatenate([[0], np.cumsum(final)])
        for b in range(2):
            s.keys[b] = k[at[b]:at[b + 1]].reshape(-1, kv, d)
            s.values[b] = v[at[b]:at[b + 1]].reshape(-1, kv, d)
        for i in range(steps):
            s.lengths = [p + (i + 1) * r for p, r in zip(past, rows)]
            want, weight, reach = ref.attention(s, query[i].double().cpu().numpy(), rows, heads, d ** -0.5)
            err = np.abs(out[i].double().cpu().numpy() - want)
            assert (err <= ref.attention_bound(s, weight, reach, want, type == N.F16)).all()
        s.lengths = final


def test_a_workspace_without_a_free_slot_is_reported(torch):
    """Sums of many blocks of an F32 chunk lie in slots that the blocks take turns with. A workspace that was not
    zeroed has none to give: the call says so and writes nothing."""
    d, heads, rows = 64, 1, 3000
    s = ref.Streams(np.random.default_rng(7), [rows] * 16, 1, d, 256)
    dev = Device(torch, s)
    starts, lengths = dev.rows([rows] * 16)
    q = torch.randn(rows * 16, d, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    ws = torch.full((native.paged_attention_workspace_bytes(dev.cache, rows * 16, rows, heads),), 1, dtype=torch.uint8,
                    device="cuda")
    out = torch.full_like(q, 7.0)

    def attend():
        torch.cuda.synchronize()
        native.call("si_paged_attention", C.byref(dev.cache), N.F32, q.data_ptr(), d, starts.data_ptr(),
                    lengths.data_ptr(), out.data_ptr(), d, rows * 16, rows, heads, 0.125, 0, ws.data_ptr(), ws.numel(),
                    None)
        torch.cuda.synchronize()

    attend()
    assert native.device_error_take(0) == 64
    assert (out == 7.0).all()
    ws.zero_()
    attend()
    assert native.device_error_take(0) == 0
    v = torch.from_numpy(np.stack([x[0, 0] for x in s.values])).cuda()  # first rows see their own token alone
    assert torch.allclose(out.view(16, rows, d)[:, 0].double(), v, rtol=1e-5, atol=0)
