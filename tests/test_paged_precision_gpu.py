"""F32 prompt chunks: the sums' truncation is made good for what a row summed, no more and no less. The unit is 2^-23
of a row's sum of p |v|; every tolerance counts the roundings that its output passes."""
import numpy as np
import pytest

import paged_reference as ref
from sharpinference_b200 import native
from test_paged_gpu import Device

pytestmark = pytest.mark.gpu
UNIT = 2.0 ** -23


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


@pytest.mark.parametrize("d", [64, 128, 192])
def test_a_row_that_sees_one_token_gets_its_values(torch, d):
    """Window 1, blocks that walk several steps. The probability as two F16 numbers: 1 unit; the sum of its two
    products, truncated: 1; the factor of the truncations, the reciprocal and three products: 2 and 0.4."""
    s = ref.Streams(np.random.default_rng(d), [1300, 700] * 20, 2, d, 64)
    rows = [300, 280] * 20
    q = np.random.default_rng(1).standard_normal((sum(rows), 2 * d)).astype(np.float32)
    got = Device(torch, s).attend(q, rows, 2, d ** -0.5, window=1)
    want = np.concatenate([v[-n:].reshape(n, -1) for v, n in zip(s.values, rows)])
    assert native.device_error_take(0) == 0
    assert (np.abs(got - want) <= 5 * UNIT * np.abs(want)).all()


@pytest.mark.parametrize("window,unmapped", [(16, False), (33, False), (0, True)])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_that_see_few_of_their_blocks_tokens(torch, d, window, unmapped):
    """Of n tokens in g runs of 16: 2 g truncated additions, n / 2 rounded ones of the probabilities (half a unit
    each), 8 units for what the other test counts and the probabilities' own roundings, and the scores' error twice."""
    streams, rows, length = 150, 40, 1000
    s = ref.Streams(np.random.default_rng(d), [length] * streams, 1, d, 64)
    if unmapped:  # only the page of the rows themselves is there
        for b in range(streams):
            for p in range((length - rows) // 64):
                s.unmap(b, p)
    q = (np.random.default_rng(2).standard_normal((streams * rows, d)) * 1e-3).astype(np.float32)
    got = Device(torch, s).attend(q, [rows] * streams, 1, d ** -0.5, window=window)
    want, weight, reach = ref.attention(s, q, [rows] * streams, 1, d ** -0.5, window)
    position = length - rows + np.tile(np.arange(rows), streams)
    first = np.maximum(position - window + 1, 0) if window else np.full_like(position, length - rows)
    n, g = position - first + 1, position // 16 - first // 16 + 1
    a = (2 * g + n / 4 + 8)[:, None] * UNIT + 2 * (d / 16 + 4) * UNIT * reach
    assert native.device_error_take(0) == 0
    assert (np.abs(got - want) <= a * weight).all()


class OneSign:
    """Keys of nearly equal weight, but one token's whose score is 8 bits above the others' where `peak` says so, and
    positive values whose channels differ by up to 2."""

    def __init__(self, seed, page_size, peak):
        self.rng, self.page_size, self.peak, self.calls = np.random.default_rng(seed), page_size, peak, 0

    def permutation(self, n):
        return self.rng.permutation(n)

    def standard_normal(self, shape):
        page, values = divmod(self.calls, 2)
        self.calls += 1
        x = self.rng.standard_normal(shape)
        if values:
            return np.abs(x) * (1 + np.arange(shape[-1]) % 32 / 32)
        x *= 1e-2
        if self.peak is not None and self.peak // self.page_size == page:
            x[:, self.peak % self.page_size] = 8 * np.log(2) / (0.1 * shape[-1] ** 0.5)
        return x


def f32(x):
    return np.asarray(x, np.float32).astype(np.float64)


def f16(x):
    return np.asarray(x, np.float16).astype(np.float64)


def place(x, bits):
    """2^-bits of the power of two below |x|."""
    return 2.0 ** (np.floor(np.log2(np.maximum(np.abs(x), 1e-30))) - bits)


def chunk_sums(score, v, every=1024):
    """Largest score, weight and sums of a row's tokens as a block of the F32 chunk kernel forms them: sum and 16 products are aligned to the largest of them, cut
    towards zero 25 places below it and their sum again 23 below itself; high halves of 64 probabilities, then low
    ones; every 1024 tokens the sums are multiplied by what the mean of the second cut loses (1 / (2 ln 2) 2^-24 for
    16 tokens) and added up rounded. score: in bits."""
    total, o, n, m = np.zeros(v.shape[1]), np.zeros(v.shape[1]), 0, score[:64].max()
    weight = 0.0

    def whole():
        return o * (1 + n * 0.72134752 * 2.0 ** -24)

    for t in range(0, len(score), 64):
        if n == every // 16:
            total, o, n = f32(total + whole()), np.zeros(v.shape[1]), 0
        top = score[t:t + 64].max()
        if top > m + 7:
            total, o, weight = (f32(x * 2.0 ** (m - top)) for x in (total, o, weight))
            m = top
        e = f32(2.0 ** (8 + score[t:t + 64] - m))
        weight += e.sum()
        high = f16(e)
        for half in (high, f16(e - high)):
            for k in range(0, len(e), 16):
                x = half[k:k + 16, None] * v[t + k:t + k + 16]
                q = place(np.maximum(np.abs(o), np.abs(x).max(0)), 25)
                o = np.trunc(o / q) * q + (np.trunc(x / q) * q).sum(0)
                q = place(o, 23)
                o = np.trunc(o / q) * q
        n += 4
    return m, weight, total + whole()


def chunk_output(score, v, cut):
    """A row's output, its tokens cut into parts of 1024 with maxima of their own or not cut."""
    step = 1024 if cut else len(score)
    parts = [chunk_sums(score[t:t + step], v[t:t + step]) for t in range(0, len(score), step)]
    m = max(p[0] for p in parts)
    weight, total = (sum(2.0 ** (p[0] - m) * p[i] for p in parts) for i in (1, 2))
    return total / weight


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("streams", [1, 90])  # tokens cut over blocks, a block for all tokens
@pytest.mark.parametrize("peak", [None, 20011])
def test_long_sums_of_one_sign_lose_what_1024_tokens_lose(torch, d, streams, peak):
    """32768 tokens (a block's, or 32 parts of 1024) of nearly equal weight whose values all add up, the case in which truncation loses most (44 units
    of a sum over 1024 tokens, of which 23 are put back; 1630 of one over all of them). The loss is compared with
    `chunk_output`, whose mean over a row's channels is the kernel's but for what rounds at random: 512 sums of the
    probabilities, off by 0.29 of a last place (0.72 units in the mean) while the sum grows, 2.7 units a row, 0.43 in
    the mean of 40 rows, and 32 sums of parts, 0.7 a value. Six times that is 3 units for the mean of all rows and 17 for a
    value, and 3 units more there for probabilities that round to the other side."""
    length, rows, ps = 32768, 40, 64
    s = ref.Streams(OneSign(d, ps, peak), [length], 1, d, ps)
    keys, values = s.keys[0][:, 0], s.values[0][:, 0]
    s.table = np.repeat(s.table, streams, 0)  # all streams on the same pages
    s.lengths = [length] * streams
    rng = np.random.default_rng(1)
    q = (0.1 + 1e-3 * rng.standard_normal((streams * rows, d))).astype(np.float32)
    got = Device(torch, s).attend(q, [rows] * streams, 1, d ** -0.5).astype(np.float64)
    assert native.device_error_take(0) == 0
    x = q.astype(np.float64) @ keys.T * d ** -0.5
    x[np.arange(length) > length - rows + np.arange(streams * rows)[:, None] % rows] = -np.inf
    p = np.exp(x - x.max(1, keepdims=True))
    want = p @ values / p.sum(1, keepdims=True)
    off, model = (got / want - 1) / UNIT, []
    for r in range(rows - 1, streams * rows, max(rows, streams * rows // 5)):
        n = length - rows + r % rows + 1
        model.append((chunk_output(x[r, :n] / np.log(2), values, streams == 1) / want[r] - 1) / UNIT)
        assert (np.abs(off[r] - model[-1]) <= 20).all()
    model = np.mean(model)
    print(f"d {d} streams {streams} peak {peak}: largest {np.abs(off).max():.1f}, mean {off.mean():.2f}, model {model:.2f}")
    assert abs(off.mean() - model) <= 3
