"""Rows of a paged call whose numbers the host only bounds: more of them in a stream than max_rows said."""
import numpy as np
import pytest

import paged_reference as ref
from sharpinference_b200 import native
from test_paged_gpu import check_attention

pytestmark = pytest.mark.gpu
N = native


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


@pytest.mark.parametrize("type", [N.F32, N.F16])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("kv,group,most", [(1, 1, 1), (2, 2, 1), (1, 3, 1), (2, 4, 1), (1, 1, 3), (1, 1, 4), (1, 5, 1),
                                           (2, 8, 4)])
def test_a_stream_of_more_rows_than_max_rows(torch, type, d, kv, group, most):
    """max_rows picks the kernel; each of them is right for any number of rows."""
    s = ref.Streams(np.random.default_rng(d + group), [40, 700, 9, 130], kv, d, 16)
    check_attention(torch, s, [1, 7, 9, 2], kv * group, type=type, most=most)
