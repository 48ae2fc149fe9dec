"""GPU: how far fp16 activations leave attention over the paged cache from 64 bits.

A value rounded to fp16 is off by 2^-11 / sqrt 3 of its binade's lower end,
2.07e-4 of itself on the average over a binade (values spread over their
logarithm: E[1 / m^2] = 0.541).  The output is rounded so, and each probability;
errors of different keys are independent, and the probabilities' weigh as the
sum itself does for values that are: sqrt 2 x 2.07e-4 = 2.93e-4 (relative L2).
K, V and the scores carry 22 bits or are exact.  Bound: 1.15 times that, for
outputs of thousands of elements; K or V rounded to fp16 as well would be 3.6e-4."""
import pytest
import torch

import paged_ref as R
from helpers import rel_l2

pytestmark = pytest.mark.gpu

BOUND = 1.15 * 2.93e-4


def attend(gb, cache, heads, kv, hd, q_lens, kv_lens, decode, scale):
    c = R.Cache(gb, cache, kv, hd, 32, kv_lens, 1)
    n = sum(q_lens)
    g = torch.Generator(device="cuda").manual_seed(2)
    q = (scale * torch.randn(n, heads * hd, generator=g, device="cuda")).half()
    out, ws = torch.empty_like(q), torch.zeros(gb.paged_workspace_bytes(heads, kv, hd, len(q_lens)), dtype=torch.uint8,
                                               device="cuda")
    cu = torch.tensor([sum(q_lens[:i]) for i in range(len(q_lens) + 1)], dtype=torch.int32, device="cuda")
    batch = gb.KVBatch(len(q_lens), n, c.len, c.table, None if decode else cu)
    (gb.paged_attention_decode if decode else gb.paged_attention_prefill)(c.h, batch, q, out, ws)
    assert gb.paged_error() == 0
    return rel_l2(out.double().cpu(), R.attention(q, c, q_lens).cpu())


@pytest.mark.parametrize("cache", [R.F16, R.Q8_0])
@pytest.mark.parametrize("hd", [64, 128])
def test_fp16_rounds_the_output_and_the_probabilities_alone(gb, cuda, cache, hd):
    assert attend(gb, cache, 32, 8, hd, [1] * 12, [40 + 150 * i for i in range(12)], True, 1.5) <= BOUND
    assert attend(gb, cache, 8, 2, hd, [300, 150], [300, 500], False, 1.5) <= BOUND


@pytest.mark.parametrize("hd", [64, 128])
def test_fp16_over_q8_0_with_scores_far_apart(gb, cuda, hd):
    """One key takes nearly all: scores of some hundreds, whose differences take
    no more than 1e-4 from their 22 bits; the output's rounding and the
    probabilities' as above."""
    for decode, q_lens, kv_lens in ((True, [1] * 9, [700, 90, 33, 500, 64, 1200, 17, 300, 128]), (False, [130, 20], [300, 20])):
        assert attend(gb, R.Q8_0, 8, 2, hd, q_lens, kv_lens, decode, 30.0) <= 4e-4
