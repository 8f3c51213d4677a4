"""Lists of si_process_logits that are allotted but still empty."""
import ctypes as C

import numpy as np
import pytest

from sharpinference_b200 import native

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


@pytest.mark.parametrize("which", ["history", "biases", "both"])
@pytest.mark.parametrize("starts", ["null", "host", "short"])
def test_an_empty_list_is_absent_whatever_its_starts_are(torch, which, starts):
    rows, vocab = 3, 1000
    x = torch.randn(rows, vocab, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    tokens, values = torch.arange(8, dtype=torch.int32, device="cuda"), torch.full((8,), 9.0, device="cuda")
    penalty = torch.full((rows,), 2.0, device="cuda")
    host, short = np.array([0, 2, 4, 6], np.int32), torch.tensor([0], dtype=torch.int32, device="cuda")
    at = {"null": None, "host": host.ctypes.data, "short": short.data_ptr()}[starts]
    c = native.LogitControls(repetition=penalty.data_ptr(), frequency=penalty.data_ptr(), presence=penalty.data_ptr())
    if which != "biases":
        c.history, c.history_starts, c.history_count = tokens.data_ptr(), at, 0
    if which != "history":
        c.bias_tokens, c.bias_values, c.bias_starts, c.bias_count = tokens.data_ptr(), values.data_ptr(), at, 0
    out, pick = torch.empty_like(x), torch.empty(rows, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    native.call("si_process_logits", native.F32, x.data_ptr(), vocab, C.byref(c), out.data_ptr(), vocab,
                pick.data_ptr(), rows, vocab, None)
    torch.cuda.synchronize()
    assert torch.equal(out, x)
    assert torch.equal(pick.long(), x.argmax(1))


@pytest.mark.parametrize("field", ["history", "bias"])
def test_starts_of_a_list_are_checked(torch, field):
    x, tokens = torch.zeros(2, 100, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    host = np.array([0, 2, 4], np.int32)
    c = native.LogitControls()
    if field == "history":
        c.history, c.history_starts, c.history_count = tokens.data_ptr(), host.ctypes.data, 4
    else:
        c.bias_tokens, c.bias_values, c.bias_starts, c.bias_count = (tokens.data_ptr(), x.data_ptr(), host.ctypes.data,
                                                                     4)
    torch.cuda.synchronize()
    for at in (host.ctypes.data, None):
        setattr(c, f"{field}_starts", at)
        assert native.lib.si_process_logits(native.F32, x.data_ptr(), 100, C.byref(c), x.data_ptr(), 100, None, 2, 100,
                                            None) == native.SI_ERR_INVALID_ARGUMENT
        assert f"{field}_starts" in native.last_error()
