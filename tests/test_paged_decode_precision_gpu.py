"""F32 decode over long streams that one warp walks whole (a batch of many): sums are truncated for 512 tokens at most,
then added up rounded."""
import numpy as np
import pytest

import paged_reference as ref
from sharpinference_b200 import native
from test_paged_gpu import Device
from test_paged_precision_gpu import UNIT, OneSign

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("streams,rows,heads", [(1900, 1, 1), (620, 1, 3), (600, 5, 2)])  # 1, 3, 10 pairs a stream
@pytest.mark.parametrize("peak", [None, 20011])
def test_long_sums_of_many_streams(torch, d, streams, rows, heads, peak):
    """32768 tokens of nearly equal weight whose values all add up. A product of 16 tokens cuts the sum and its own terms
    towards zero, each by less than 2^-25 of the largest and their sum by less than 2^-23: 17 / 4 + 1 units of the sum so
    far at most, half of that in the mean. 512 tokens make 32 products (64 where both halves of the probabilities go into
    one accumulator) of a sum that grows from nothing: 84 (168) units at most, half of it in the mean. 64 rounded additions
    of half a unit each and the sums of the probabilities: 40 more. Without the rest every 512 tokens 1030 (880) are lost."""
    length, ps = 32768, 64
    s = ref.Streams(OneSign(d, ps, peak), [length], 1, d, ps)
    keys, values = (torch.from_numpy(x[0][:, 0]).cuda() for x in (s.keys, s.values))
    s.table = np.repeat(s.table, streams, 0)  # all streams on the same pages
    s.lengths = [length] * streams
    rng = np.random.default_rng(1)
    q = (0.1 + 1e-3 * rng.standard_normal((streams * rows, heads, d))).astype(np.float32)
    got = Device(torch, s).attend(q.reshape(streams * rows, -1), [rows] * streams, heads, d ** -0.5)
    got = torch.from_numpy(got).cuda().double().view(streams, rows, heads, d)
    assert native.device_error_take(0) == 0
    q = torch.from_numpy(q).cuda().double().view(streams, rows, heads, d)
    off = []
    for b in range(0, streams, streams // 30):
        for i in range(rows):
            x = (q[b, i] @ keys.T * d ** -0.5)[:, :length - rows + i + 1]
            off.append(got[b, i] / (torch.softmax(x, 1) @ values[:length - rows + i + 1]) - 1)
    off = torch.stack(off) / UNIT
    once = 84 if rows * heads <= 4 else 168
    print(f"d {d} pairs {rows * heads} peak {peak}: largest {off.abs().max():.1f}, mean {off.mean():.2f} units")
    assert off.abs().max() <= once + 40
    assert off.mean().abs() <= once / 2 + 5


def test_long_sums_whose_maxima_move(torch):
    """Scores that rise from token to token, so that put away sums are scaled: against the bound of any row."""
    d, ps, length, streams = 128, 64, 3000, 900

    class Rising:
        def __init__(self):
            self.rng, self.calls = np.random.default_rng(5), 0

        def permutation(self, n):
            return self.rng.permutation(n)

        def standard_normal(self, shape):
            self.calls += 1
            return self.rng.standard_normal(shape) * (1 + 0.05 * self.calls)

    s = ref.Streams(Rising(), [length], 1, d, ps)
    s.table, s.lengths = np.repeat(s.table, streams, 0), [length] * streams
    for rows, heads in ((1, 3), (2, 4)):
        q = np.random.default_rng(rows).standard_normal((streams * rows, heads * d)).astype(np.float32)
        got = Device(torch, s).attend(q, [rows] * streams, heads, d ** -0.5)
        one = ref.Streams.__new__(ref.Streams)
        one.__dict__.update(s.__dict__)
        one.keys, one.values = s.keys * 4, s.values * 4
        few = [0, 1, streams // 2, streams - 1]
        one.lengths, one.mapped = [length] * 4, s.mapped[:1].repeat(4, 0)
        pick = np.concatenate([np.arange(b * rows, b * rows + rows) for b in few])
        want, weight, reach = ref.attention(one, q[pick], [rows] * 4, heads, d ** -0.5)
        assert (np.abs(got[pick] - want) <= ref.attention_bound(one, weight, reach, want, False)).all()


def test_long_sums_of_many_f16_streams(torch):
    """131072 tokens, sums put away every 8192: 512 products lose at most 5.25 units each of a sum that grows from nothing,
    672 in the mean; probabilities round by up to 2^-11, a quarter of that in the mean of many."""
    d, streams, length, ps = 128, 1900, 131072, 256
    s = ref.Streams(OneSign(d, ps, None), [length], 1, d, ps)
    keys, values = (torch.from_numpy(x[0][:, 0]).cuda() for x in (s.keys, s.values))
    s.table, s.lengths = np.repeat(s.table, streams, 0), [length] * streams
    q = (0.1 + 1e-3 * np.random.default_rng(1).standard_normal((streams, d))).astype(np.float16)
    got = torch.from_numpy(Device(torch, s).attend(q, [1] * streams, 1, d ** -0.5, type=native.F16)).cuda().double()
    few = torch.arange(0, streams, 90, device="cuda")
    x = torch.from_numpy(q.astype(np.float64)).cuda()[few] @ keys.T * d ** -0.5
    off = got[few] / (torch.softmax(x, 1) @ values) - 1
    print(f"mean {off.mean():.2e}, largest {off.abs().max():.2e}")
    assert off.mean().abs() <= 672 * UNIT + 2.0 ** -13
