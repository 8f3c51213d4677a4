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
