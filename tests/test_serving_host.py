"""CPU: what examples/serve_batch.py's server admits."""
import os
import sys

import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.fixture
def server():
    import serve_batch as ex
    s = ex.Server.__new__(ex.Server)   # without a model's memory

    class Model:
        max_seq = 100
    s.m, s.page, s.max_running, s.free, s.waiting, s.running = Model(), 16, 4, list(range(6)), [], []
    return ex, s


def test_requests_that_cannot_be_answered(server):
    """No prompt (its logits would be another request's), no token wanted, longer than the cache."""
    ex, s = server
    for prompt, n_new in (([], 4), ([1, 2], 0), ([1, 2], -1), ([1] * 90, 11), ([1] * 95, 5)):
        with pytest.raises(ValueError):
            s.submit(ex.Request(prompt, n_new))
    assert not s.waiting
    s.submit(ex.Request([1], 1))
    s.submit(ex.Request([1] * 90, 6))
    assert len(s.waiting) == 2
