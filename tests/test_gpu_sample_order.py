"""GPU: batches whose rows gb_sample takes in another order (more than run at
once, few against the vocabulary), and those beside the rule's borders."""
import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,vocab", [(37, 50001), (38, 50001), (62, 50001), (63, 50001), (61, 128256), (148, 128256),
                                     (149, 128256)])
def test_a_batch_gives_each_row_the_token_it_has_alone(gb, cuda, n, vocab):
    g = torch.Generator(device="cuda").manual_seed(n)
    logits = 2.0 * torch.randn(n, vocab, generator=g, device="cuda")
    i = torch.arange(n)
    t = torch.where(i % 5 == 0, 0.0, 0.9)
    k = torch.where(i % 5 % 2 == 0, 40, torch.where(i % 7 == 3, 700, 0)).int()
    p, m = torch.where(i % 5 >= 3, 0.9, 1.0), torch.where(i % 5 == 4, 0.05, 0.0)
    u = (i * 0.37 + 0.05) % 1.0
    a = [x.cuda() for x in (u, t, k, p, m)]
    out = torch.full((n,), -9, dtype=torch.int32, device="cuda")
    gb.sample(logits, out, *a)
    alone = torch.full((n,), -9, dtype=torch.int32, device="cuda")
    for r in range(n):
        gb.sample(logits[r: r + 1], alone[r: r + 1], *(x[r: r + 1] for x in a))
    assert torch.equal(out, alone)
    for r in range(0, n, 12):
        assert out[r].item() == R.sample_row(logits[r], t[r].item(), k[r].item(), p[r].item(), m[r].item(), u[r].item())
