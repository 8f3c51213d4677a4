"""The serving example with a pool that does not hold all requests at once."""
import numpy as np
import pytest

from sharpinference_b200 import native, phi4

pytestmark = pytest.mark.gpu
CFG = dict(phi4.TINY, context=400, vocab=384, weight_type=native.F16, embedding_type=native.F16)


@pytest.fixture(scope="module")
def serving():
    pytest.importorskip("torch")
    import examples.paged_serving as module
    return module


def _server(serving, slots, pages):
    return serving.PagedServer(CFG, serving.random_model(CFG, 1), slots, pages=pages, page_size=32, chunk=70)


def _requests(serving):
    rng = np.random.default_rng(2)
    return [serving.Request(rng.integers(0, CFG["vocab"], n).astype(np.int32), new)
            for n, new in [(90, 40), (30, 3), (100, 60), (1, 1), (64, 33), (10, 150)]]


def test_a_small_pool_serves_the_same_tokens_one_after_the_other(serving):
    want = _requests(serving)
    wide = _server(serving, 6, 64)
    for r in want:
        wide.submit(r)
    wide.run()
    got = _requests(serving)
    small = _server(serving, 3, 6)  # the largest requests take 5 pages each
    for r in got:
        small.submit(r)
    small.run()
    assert [len(r.tokens) for r in got] == [r.new_tokens for r in got]
    # single rows and chunks of other sizes round differently: the first tokens of each request are far from ties
    assert [r.tokens[0] for r in got] == [r.tokens[0] for r in want]
    assert sorted(small.free) == list(range(6)) and (small.table == -1).all()


def test_requests_that_can_not_be_served_are_refused(serving):
    server = _server(serving, 2, 4)
    prompt = np.arange(10, dtype=np.int32)
    for new in (0, -3):
        with pytest.raises(native.ArgumentError):
            server.submit(serving.Request(prompt, new))
    with pytest.raises(native.ArgumentError):
        server.submit(serving.Request(prompt, 130))  # 139 tokens in the cache, the pool holds 128
    server.submit(serving.Request(prompt, 119))
    server.run()
