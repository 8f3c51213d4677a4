"""F32 rows that one token owns: channels in which its value is 0 are made of the others' probabilities, however small,
and what that takes does not grow out of proportion."""
import ctypes as C

import numpy as np
import pytest

import paged_reference as ref
from sharpinference_b200 import native
from test_paged_gpu import Device

pytestmark = pytest.mark.gpu
N = native


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


def check(s, query, rows, heads, got, window=0):
    """F16 probabilities hold 2^-33 of the largest that they are summed with. In a row in which all other tokens are
    together below 2^-16 of one (2^-18 here: the kernels' sums are rounded) that is the largest of the others."""
    want, weight, reach = ref.attention(s, query, rows, heads, s.d ** -0.5, window)
    bound, r = ref.attention_bound(s, weight, reach, want, False), 0
    floor, group = np.zeros_like(bound).reshape(-1, heads, s.d), heads // s.kv
    q = np.asarray(query, np.float64).reshape(-1, heads, s.d)
    owned = 0
    for b, n in enumerate(rows):
        for i in range(n):
            p = s.lengths[b] - n + i
            t = np.arange(max(0, p - window + 1) if window else 0, p + 1)
            t = t[s.mapped[b][t // s.page_size]] if t.size else t
            for h in range(heads if t.size else 0):
                x = s.d ** -0.5 * (s.keys[b][t, h // group] @ q[r, h])
                e = np.sort(np.exp(x - x.max()))
                others = e[:-1].sum()
                owned += 0 < others < 2.0 ** -18
                floor[r, h] = 2.0 ** -33 * (others if others < 2.0 ** -18 else 1) * np.abs(s.values[b][t, h // group]).sum(0)
            r += 1
    assert native.device_error_take(0) == 0
    err = np.abs(got - want)
    assert (err <= bound + floor.reshape(bound.shape)).all(), np.max(err / (bound + floor.reshape(bound.shape)))
    return owned


@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("spread", [8, 30])
@pytest.mark.parametrize("rows,lengths", [([1, 1, 2], [300, 17, 900]), ([5, 6], [60, 1500]), ([20, 33], [700, 41]),
                                          ([150, 40, 1], [420, 40, 300]), ([60], [1700])])
def test_peaked_rows(torch, d, spread, rows, lengths):
    s = ref.Streams(np.random.default_rng(d), lengths, 1, d, 32)
    q = (np.random.default_rng(spread).standard_normal((sum(rows), 4 * d)) * spread).astype(np.float32)
    assert check(s, q, rows, 4, Device(torch, s).attend(q, rows, 4, d ** -0.5)) > 0 or spread < 30


def test_window_and_unmapped_pages_of_owned_rows(torch):
    for rows, lengths in (([1, 2], [300, 517]), ([40, 90], [700, 300])):
        s = ref.Streams(np.random.default_rng(1), lengths, 2, 128, 32)
        s.unmap(0, 2), s.unmap(0, 5), s.unmap(1, 8)
        for window in (0, 20, 150):
            q = (np.random.default_rng(window).standard_normal((sum(rows), 512)) * 50).astype(np.float32)
            got = Device(torch, s).attend(q, rows, 4, 128 ** -0.5, window)
            assert check(s, q, rows, 4, got, window) > 0


def test_a_value_that_is_not_finite_in_owned_rows(torch):
    for rows, length in ((1, 200), (40, 260), (40, 2000)):
        d, token = 128, length - rows - 20
        s = ref.Streams(np.random.default_rng(2), [length], 1, d, 16)
        q = (np.random.default_rng(3).standard_normal((rows, 2 * d)) * 1e4).astype(np.float32)
        clean = Device(torch, s).attend(q, [rows], 2, d ** -0.5)
        page, slot, group = s.table[0, token // 16], token % 16, 1
        s.pool[page, 17 * d + (group * 16 + slot) * 2:][:2] = 0xFF
        got = Device(torch, s).attend(q, [rows], 2, d ** -0.5).reshape(rows, 2, d)
        want = clean.reshape(rows, 2, d).copy()
        want[:, :, 32:64] = np.nan
        assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("rows,length", [(16, 16384), (300, 2000), (1, 16384)])
def test_owned_rows_do_not_take_out_of_proportion(torch, rows, length):
    """Against the same call with ordinary scores: a few walks over the tokens more for eight rows together (measured 4
    to 35 times), not one for each row by itself (200 to 2800 times)."""
    d, heads, kv, ps = 128, 8, 2, 64
    s = ref.Streams(np.random.default_rng(4), [length], kv, d, ps)
    dev = Device(torch, s)
    starts, lengths = dev.rows([rows])
    q = torch.randn(rows, heads * d, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    peaked = q * 300
    out = torch.empty_like(q)
    ws = torch.zeros(native.paged_attention_workspace_bytes(dev.cache, rows, rows, heads), dtype=torch.uint8, device="cuda")

    def time(x):
        best = 1e9
        for _ in range(4):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            native.call("si_paged_attention", C.byref(dev.cache), N.F32, x.data_ptr(), heads * d, starts.data_ptr(),
                        lengths.data_ptr(), out.data_ptr(), heads * d, rows, rows, heads, d ** -0.5, 0, ws.data_ptr(),
                        ws.numel(), torch.cuda.current_stream().cuda_stream)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    assert time(peaked) <= 100 * time(q)
