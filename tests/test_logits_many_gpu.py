"""si_process_logits of many rows: clusters of 8, 4, 2 and 1 blocks to a row, with one chunk and with several."""
import numpy as np
import pytest

from sharpinference_b200 import native
from test_logits_gpu import Case, same

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


@pytest.mark.parametrize("type", [native.F32, native.F16])
@pytest.mark.parametrize("rows,vocab", [(20, 16384), (20, 70001), (37, 33000), (49, 140000), (74, 20005), (100, 17000),
                                        (128, 40004), (148, 8193), (149, 20000), (300, 9001), (600, 2000)])
def test_many_rows_equal_the_definition(torch, type, rows, vocab):
    case = Case(np.random.default_rng(vocab + rows), rows, vocab, type, history=700, biases=40, mask="some")
    want = case.want()
    same(case.run(torch), want)
    same(case.run(torch, in_place=True, pad=3), want)
