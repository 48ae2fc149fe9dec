"""GPU: the batched-serving operators together, as examples/serve_batch.py uses
them: packed prompts, single-token steps, sampling, pages changing hands."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ex(gb, cuda):
    import serve_batch
    return serve_batch


def prompts(n, seed, most=150):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 1000, (int(torch.randint(1, most, (1,), generator=g)),), generator=g).tolist()
            for _ in range(n)]


@pytest.mark.parametrize("cache", ["q8_0", "f16"])
def test_a_step_continues_the_prompt(gb, ex, cache):
    """Logits of a single-token step after a prompt against those of the prompt
    one token longer, run whole: the same cache values, the same sums in
    another order (1e-4 after two layers and the head)."""
    model = ex.Decoder()
    ct = gb.DT_Q8_0 if cache == "q8_0" else gb.DT_F16
    p = prompts(1, 3)[0] + [7, 8]
    a, b = ex.Server(model, cache_type=ct), ex.Server(model, cache_type=ct)
    ra, rb = ex.Request(p[:-1], 4), ex.Request(p, 4)
    for s, r in ((a, ra), (b, rb)):
        r.pages = [s.free.pop() for _ in range(12)]
    a._run([ra], ra.prompt, [len(ra.prompt)])
    ra.tokens[-1] = p[-1]
    la = a._run([ra], [p[-1]], [1])
    lb = b._run([rb], rb.prompt, [len(rb.prompt)])
    assert gb.paged_error() == 0
    assert ((la - lb).norm() / lb.norm()).item() <= 1e-4


@pytest.mark.parametrize("cache", ["q8_0", "f16"])
def test_batched_answers_are_those_of_each_alone(gb, ex, cache):
    model = ex.Decoder()
    ct = gb.DT_Q8_0 if cache == "q8_0" else gb.DT_F16
    settings = [dict(), dict(temperature=0.8, top_k=5), dict(temperature=0.7, top_p=0.5), dict(temperature=0.5, min_p=0.2)]

    def requests():
        return [ex.Request(p, 6, seed=i, **settings[i % 4]) for i, p in enumerate(prompts(9, 5))]

    together = requests()
    server = ex.Server(model, n_pages=40, cache_type=ct, max_running=5)   # some have to wait for pages
    for r in together:
        server.submit(r)
    server.run()
    assert sorted(server.free) == list(range(40))
    for r, alone in zip(together, requests()):
        s = ex.Server(model, n_pages=40, cache_type=ct)
        s.submit(alone)
        s.run()
        assert len(r.tokens) == 6 and r.tokens == alone.tokens
