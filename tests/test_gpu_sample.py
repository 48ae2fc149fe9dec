"""GPU: gb_sample against its definition in Python integers: every token is
equal, whatever the batch."""
import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu


def draw(gb, logits, u, t=None, k=None, p=None, m=None):
    n = logits.shape[0]
    f = lambda v, dt=torch.float32: None if v is None else torch.tensor(v, dtype=dt, device="cuda")  # noqa: E731
    out = torch.full((n,), -9, dtype=torch.int32, device="cuda")
    gb.sample(logits, out, f(u), f(t), f(k, torch.int32), f(p), f(m))
    return out.tolist()


def expect(logits, u, t=None, k=None, p=None, m=None):
    n = logits.shape[0]
    at = lambda v, i, d: d if v is None else v[i]  # noqa: E731
    uf = torch.tensor(u, dtype=torch.float32).tolist()
    return [R.sample_row(logits[i], at(t, i, 1.0), at(k, i, 0), at(p, i, 1.0), at(m, i, 0.0), uf[i]) for i in range(n)]


def rows(n, vocab, seed, scale=2.0, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.full((n, vocab + pad), float("inf"), device="cuda")
    x[:, :vocab] = scale * torch.randn(n, vocab, generator=g, device="cuda")
    return x[:, :vocab]


SETTINGS = [
    dict(),
    dict(t=0.7),
    dict(t=1.3, k=5),
    dict(k=1),
    dict(p=0.9),
    dict(p=0.0),
    dict(t=0.5, p=0.3),
    dict(m=0.1),
    dict(m=1.0),
    dict(t=0.8, k=40, p=0.95, m=0.05),
    dict(t=2.0, k=100000, p=0.999),
    dict(t=0.0),
    dict(t=1e-30),
    dict(t=50.0, p=0.5),
]


@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 1025, 32000, 128256])
def test_against_the_definition(gb, cuda, vocab):
    us = [0.0, 0.1, 0.37, 0.5, 0.83, 0.9999999]
    n = len(SETTINGS) * len(us)
    logits = rows(n, vocab, vocab, pad=3)
    each = [(s, u) for s in SETTINGS for u in us]
    args = dict(t=[s.get("t", 1.0) for s, _ in each], k=[s.get("k", 0) for s, _ in each],
                p=[s.get("p", 1.0) for s, _ in each], m=[s.get("m", 0.0) for s, _ in each])
    u = [u for _, u in each]
    got = draw(gb, logits, u, **args)
    assert got == expect(logits, u, **args)
    # a row drawn alone gives the same token
    for i in range(0, n, 17):
        assert draw(gb, logits[i: i + 1], u[i: i + 1], **{a: v[i: i + 1] for a, v in args.items()}) == [got[i]]
    assert draw(gb, logits, u) == expect(logits, u)   # no parameter arrays


@pytest.mark.parametrize("vocab", [7, 4096, 50001])
def test_ties_masks_and_odd_values(gb, cuda, vocab):
    inf, nan = float("inf"), float("nan")
    x = rows(12, vocab, 3)
    x[0] = 1.5                                   # all equal
    x[1] = torch.round(x[1])                     # many ties
    x[2] = -inf                                  # nothing left
    x[3] = nan
    x[4, : vocab - 1] = -inf                     # one left, the last
    x[5, vocab // 2] = inf                       # certain
    x[6] = inf
    x[7, ::2] = nan
    x[8, 1::2] = -inf
    x[9] = torch.where(x[9] > 0, 0.0, -0.0)      # zeros of both signs are equal
    x[10] = torch.finfo(torch.float32).min                        # the type's lowest
    x[10, vocab - 1] = 0
    x[11] = 3e38 * torch.sign(x[11])
    for s in SETTINGS:
        for u in (0.0, 0.42, 0.77):
            a = {n: [v] * 12 for n, v in s.items()}
            got = draw(gb, x, [u] * 12, **a)
            assert got == expect(x, [u] * 12, **a), (s, u)
            assert got[2] == got[3] == -1 and got[4] == vocab - 1 and got[5] == vocab // 2


def test_lowest_index_of_equal_logits(gb, cuda):
    x = torch.zeros(1, 5000, device="cuda")
    x[0, [17, 900, 4999]] = 1.0
    assert draw(gb, x, [0.99], t=[0.0]) == [17]
    assert draw(gb, x, [0.99], k=[1]) == [17]
    assert draw(gb, x, [0.99], k=[2]) == [900]
    assert draw(gb, x, [0.99], p=[0.0]) == [17]
    assert draw(gb, x, [0.99], k=[5]) == [4999] and draw(gb, x, [0.999], k=[4], t=[100.0]) == [4999]


def test_parameters_out_of_range_and_the_largest_vocabulary(gb, cuda):
    nan = float("nan")
    x = rows(6, 262144, 8)
    a = dict(t=[1.0, nan, -1.0, 1.0, 1.0, 1.0], k=[-3, 0, 0, 0, 1 << 30, 0], p=[1.0, 1.0, 1.0, 7.0, nan, -2.0],
             m=[nan, 0.0, 0.0, -1.0, 0.0, 9.0])
    u = [0.3, 0.3, 0.3, 1.0, -4.0, nan]
    fixed = dict(t=[1.0, 0.0, 0.0, 1.0, 1.0, 1.0], k=[0] * 6, p=[1.0, 1.0, 1.0, 1.0, 1.0, 0.0], m=[0.0] * 6)
    assert draw(gb, x, u, **a) == expect(x, [0.3, 0.3, 0.3, 0.99999999, 0.0, 0.0], **fixed)


def test_frequencies(gb, cuda):
    """Draws over an even grid of u: each token as often as its probability says."""
    p = torch.tensor([0.5, 0.25, 0.125, 0.0625, 0.0625], device="cuda")
    n = 4096
    x = p.log().expand(n, 5).contiguous()
    u = ((torch.arange(n) + 0.5) / n).tolist()
    got = torch.bincount(torch.tensor(draw(gb, x, u)), minlength=5) / n
    # a boundary of the running sum moves at most one grid point
    assert (got - p.cpu()).abs().max() <= 2.0 / n


@pytest.mark.parametrize("vocab", [5, 3001])
def test_infinite_temperature(gb, cuda, vocab):
    """Every token that is not masked weighs the same; a masked one nothing."""
    logits = rows(6, vocab, 9)
    logits[:, ::3] = float("-inf")
    left = [i for i in range(vocab) if i % 3]
    u = [0.0, 0.2, 0.5, 0.7, 0.9, 0.99]
    want = [left[int(len(left) * torch.tensor(v).mul(2**24).floor().item() / 2**24)] for v in u]
    assert draw(gb, logits, u, [float("inf")] * 6) == want
    assert draw(gb, logits, u, [float("inf")] * 6, k=[vocab - 1] * 6, p=[1.0] * 6) == want
    # nucleus of equal weights: the largest logits, ties by index
    half = draw(gb, logits, u, [float("inf")] * 6, p=[0.5] * 6)
    for r, tok in enumerate(half):
        order = sorted(left, key=lambda i: (-logits[r, i].item(), i))
        kept = sorted(order[: -(-len(left) // 2)])
        assert tok == kept[int(len(kept) * torch.tensor(u[r]).mul(2**24).floor().item() / 2**24)]


@pytest.mark.parametrize("n", [38, 61, 148, 149])
def test_batches_of_different_rows(gb, cuda, n):
    """More rows than run at once are taken in another order; each row's token
    is the one that it gives alone."""
    logits = rows(n, 5003, n)
    u = [(i * 0.37 + 0.05) % 1.0 for i in range(n)]
    t, k = [0.0 if i % 5 == 0 else 0.9 for i in range(n)], [40 if i % 5 in (2, 4) else 700 if i % 7 == 3 else 0 for i in range(n)]
    p, m = [0.9 if i % 5 >= 3 else 1.0 for i in range(n)], [0.05 if i % 5 == 4 else 0.0 for i in range(n)]
    got = draw(gb, logits, u, t, k, p, m)
    assert got == expect(logits, u, t, k, p, m)
    assert got == [draw(gb, logits[i:i + 1], u[i:i + 1], t[i:i + 1], k[i:i + 1], p[i:i + 1], m[i:i + 1])[0] for i in range(n)]
