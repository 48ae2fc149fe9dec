"""GPU: attention over the paged cache where q, K or V hold NaN, infinities or
values past fp16's range: the rows and columns that are no number or infinite
are those of the definition, and every other one is as exact as ever.

The definition: a token's softmax and sum run over the positions that it sees
and no others, so what stands at a later position never reaches it.  An output
element is finite in the kernel where it is in 64 bits (rounded to the output's
type).

Tolerances (L2 of a row against its own size), derived as for finite values:
F32 activations 22 significant bits of q and of the probabilities, 3e-5; F16
activations the output's rounding and the probabilities' (2^-11 / sqrt 3 =
2.8e-4 each, 4e-4 together) and a factor of 3 for a single row, 1.2e-3."""
import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")
F32, F16 = torch.float32, torch.float16
TOL = {F32: 3e-5, F16: 1.2e-3}
ACT = {"f32": F32, "f16": F16}
CACHE = {"f16": R.F16, "q8_0": R.Q8_0}


def cu_of(q_lens):
    return torch.tensor([sum(q_lens[:i]) for i in range(len(q_lens) + 1)], dtype=torch.int32, device="cuda")


def definition(q, c, q_lens):
    """fp64 [tokens][heads * hd], over the seen positions alone."""
    out, t0, hd, kv = [], 0, c.hd, c.n_kv
    for s, n in enumerate(q_lens):
        m = c.kv_lens[s]
        x = q[t0: t0 + n].double().reshape(n, kv, -1, 1, hd)
        t0 += n
        k, v = (c.get(p, s, m).transpose(0, 1) for p in c.pools)       # [kv][m][hd]
        o = torch.zeros(n, kv, x.shape[2], hd, dtype=torch.float64, device="cuda")
        for i in range(n):
            see = m - n + i + 1
            if see > 0:
                sc = (x[i] * k[:, None, :see]).sum(-1) / hd ** 0.5       # [kv][group][see]
                p = torch.softmax(sc, -1)
                o[i] = (p[..., None] * v[:, None, :see]).sum(-2)
        out.append(o.reshape(n, -1))
    return torch.cat(out)


def check(gb, c, q, q_lens, decode, what=""):
    hd = c.hd
    heads = q.shape[1] // hd
    out = torch.full_like(q, 3.0)
    ws = torch.zeros(gb.paged_workspace_bytes(heads, c.n_kv, hd, len(q_lens)), dtype=torch.uint8, device="cuda")
    batch = gb.KVBatch(len(q_lens), sum(q_lens), c.len, c.table, None if decode else cu_of(q_lens))
    (gb.paged_attention_decode if decode else gb.paged_attention_prefill)(c.h, batch, q, out, ws)
    ref = definition(q, c, q_lens)
    there = torch.isfinite(ref.to(q.dtype))
    wrong = (torch.isfinite(out) != there).nonzero()
    assert not len(wrong), (what, len(wrong), wrong[:4].tolist())
    # a head's row by itself, against its own size (in 64 bits: a column may pass the output's type)
    err = torch.where(there, out.double() - ref, 0.0).unflatten(1, (heads, hd)).norm(dim=-1)
    size = torch.where(torch.isfinite(ref), ref, 0.0).unflatten(1, (heads, hd)).norm(dim=-1)
    assert (err <= TOL[q.dtype] * size).all(), (what, (err / size.clamp(min=1e-300)).max().item())
    # the workspace is ready for the next call, and fit for finite rows
    again = torch.empty_like(out)
    (gb.paged_attention_decode if decode else gb.paged_attention_prefill)(c.h, batch, q, again, ws)
    assert torch.equal(torch.nan_to_num(again, nan=5.0), torch.nan_to_num(out, nan=5.0)), what
    assert gb.paged_error() == 0


def rows(n, width, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (1.5 * torch.randn(n, width, generator=g, device="cuda")).to(dtype)


def put_value(c, pool, s, pos, head, col, value):
    """A value (for Q8_0 its block's scale) in the cache."""
    pg, r = c.table[s, pos // c.page].item(), pos % c.page
    halves, scales = c.parts(pool)
    if scales is not None:
        scales[pg, head, r, col // 32] = value
    else:
        halves[pg, head, r, col] = value


FORMS = [(a, c, hd) for a in ("f32", "f16") for c in ("f16", "q8_0") for hd in (64, 128)]


# ------------------------------------------------------------------ single tokens
@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("kv_len,some", [(40, 20), (300, 299)])
def test_decode_scores_of_minus_infinity(gb, cuda, act, kv_len, some):
    """Keys whose score is -inf weigh nothing, for heads that see finite ones
    beside them and next to heads that do not."""
    minus_infinity(gb, act, kv_len, some, True, 1)


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("kv_len,some", [(3000, 2500), (20011, 17000)])
def test_decode_ctas_with_scores_of_minus_infinity_alone(gb, cuda, act, kv_len, some):
    minus_infinity(gb, act, kv_len, some, True, 1)


def minus_infinity(gb, act, kv_len, some, decode, n):
    hd = 64
    c = R.Cache(gb, R.F16, 1, hd, 64, [kv_len], 7)
    pos = torch.arange(kv_len, device="cuda")
    pages, at = c.table[0, pos // 64].long(), pos % 64
    halves, _ = c.parts(c.pools[0])
    halves[pages[:some], 0, at[:some], 9] = INF
    q = rows(n, 8 * hd, ACT[act], 8)
    q[:, 9::hd] = -q[:, 9::hd].abs() - 0.1
    check(gb, c, q, [n], decode, "the first keys")
    q[:, 9 + 3 * hd] *= -1                     # +inf for head 3 alone: no number
    check(gb, c, q, [n], decode, "head 3")
    q[:, 9 + 3 * hd] = 0.0                     # 0 x inf: no number either
    check(gb, c, q, [n], decode, "head 3, zero")
    halves[pages, 0, at, 11] = INF             # -inf at every position, but for head 5
    q[:, 11::hd] = -q[:, 11::hd].abs() - 0.1
    q[:, 9 + 3 * hd] = -0.25
    check(gb, c, q, [n], decode, "nothing left")
    halves[pages, 0, at, 9] = 0.25             # head 5: +inf at every position
    q[:, 11 + 5 * hd] *= -1
    check(gb, c, q, [n], decode, "nothing left, head 5")


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("act,hd", [(a, hd) for a in ("f32", "f16") for hd in (64, 128)])
def test_decode_in_an_f16_cache_at_every_place(gb, cuda, act, hd, value, which):
    """K (0) or V (1) at every position modulo 16."""
    every_place(gb, act, "f16", hd, value, which, True)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("act,hd", [(a, hd) for a in ("f32", "f16") for hd in (64, 128)])
def test_decode_in_a_q8_0_cache_at_every_place(gb, cuda, act, hd, which):
    """A block's scale (an append writes finite ones)."""
    every_place(gb, act, "q8_0", hd, NAN, which, True)


def every_place(gb, act, cache, hd, value, which, decode):
    n = 1 if decode else 64
    q = rows(64, 4 * hd, ACT[act], 4)[:n]
    for pos in list(range(64, 80)) + [0, 98]:
        c = R.Cache(gb, CACHE[cache], 2, hd, 32, [99], pos)
        put_value(c, c.pools[which], 0, pos, pos % 2, (7 * pos) % hd, value)
        check(gb, c, q, [n], decode, pos)


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("kv_lens", [[99], [2000], [99] * 400])
def test_decode_an_infinite_value_that_weighs_next_to_nothing(gb, cuda, act, kv_lens):
    """A key hundreds of units below the maximum, in a warp that sees the
    maximum or another: in 64 bits its infinite value still is one."""
    c = R.Cache(gb, R.F16, 1, 64, 32, kv_lens, 4)
    n, m = len(kv_lens), kv_lens[0]
    q = rows(n, 64, ACT[act], 4)
    for s in range(n):
        x = torch.zeros(m, 1, 64, device="cuda")
        x[m - 1, 0] = 400 * q[s].float() / q[s].float().norm()
        c.put(c.pools[0], s, x)
        put_value(c, c.pools[1], s, (37 * s) % (m - 1), 0, 40, INF)
    check(gb, c, q, [1] * n, True)


@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("act,cache,hd", FORMS)
def test_decode_in_q(gb, cuda, act, cache, hd, value):
    """One query head's row, and no other."""
    in_q(gb, act, cache, hd, value, True, [1, 1])


def in_q(gb, act, cache, hd, value, decode, q_lens):
    c = R.Cache(gb, CACHE[cache], 2, hd, 16, [100, 37], 1)
    q = rows(sum(q_lens), 4 * hd, ACT[act], 2)
    q[sum(q_lens) - 1, hd + 5] = value
    q[0, 3 * hd - 1] = value
    check(gb, c, q, q_lens, decode)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_decode_q8_0_beyond_the_largest_half(gb, cuda, act, hd, which):
    """An append's scale reaches 65504, its values 127 times that: they are finite."""
    beyond(gb, act, hd, which, True)


def beyond(gb, act, hd, which, decode):
    n = 1 if decode else 64
    for pos, size in ((5, 7e4), (60, 3e5), (70, 5e6), (98, 1e5)):
        c = R.Cache(gb, R.Q8_0, 2, hd, 32, [99], pos)
        x = torch.randn(99, 2, hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(pos))
        x[pos, 1, 3::5] = size
        c.put(c.pools[which], 0, x)
        check(gb, c, rows(n, 4 * hd, ACT[act], 4), [n], decode, pos)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("cache,value", [("f16", NAN), ("f16", INF), ("q8_0", NAN)])
@pytest.mark.parametrize("act", ["f32", "f16"])
def test_decode_over_a_long_axis(gb, cuda, act, cache, value, which):
    """Keys split over CTAs and joined."""
    long_axis(gb, act, cache, value, which, True, 1)


def long_axis(gb, act, cache, value, which, decode, n):
    for pos in (3, 2990):
        c = R.Cache(gb, CACHE[cache], 1, 128, 64, [3000], 6)
        put_value(c, c.pools[which], 0, pos, 0, 77, value)
        check(gb, c, rows(n, 4 * 128, ACT[act], 5), [n], decode, pos)


# ------------------------------------------------------------------ packed prompts
@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("act,cache,hd", FORMS)
def test_prefill_in_q(gb, cuda, act, cache, hd, value):
    in_q(gb, act, cache, hd, value, False, [100, 9])


@pytest.mark.parametrize("act,cache,hd", FORMS)
def test_prefill_no_number_in_k_at_every_place(gb, cuda, act, cache, hd):
    every_place(gb, act, cache, hd, NAN, 0, False)


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("cache", ["f16", "q8_0"])
def test_prefill_no_number_in_k_over_a_long_axis(gb, cuda, act, cache):
    long_axis(gb, act, cache, NAN, 0, False, 16)


@pytest.mark.parametrize("value", [INF, -INF])
@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_prefill_infinite_k_at_every_place(gb, cuda, act, hd, value):
    every_place(gb, act, "f16", hd, value, 0, False)


@pytest.mark.parametrize("cache,value", [("f16", NAN), ("f16", INF), ("f16", -INF), ("q8_0", NAN)])
@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_prefill_in_v_at_every_place(gb, cuda, act, cache, hd, value):
    """Rows that do not see the position are as if it were not there."""
    every_place(gb, act, cache, hd, value, 1, False)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_prefill_q8_0_beyond_the_largest_half(gb, cuda, act, hd, which):
    """Finite values, and those of later tokens leave earlier rows alone."""
    beyond(gb, act, hd, which, False)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("cache,value", [("f16", NAN), ("f16", INF), ("q8_0", NAN)])
@pytest.mark.parametrize("act", ["f32", "f16"])
def test_prefill_few_rows_over_a_long_axis(gb, cuda, act, cache, value, which):
    """Keys split over CTAs and joined: a value early, and one that only the last rows see."""
    long_axis(gb, act, cache, value, which, False, 16)


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("kv_len,some", [(40, 20), (300, 280), (3000, 2500)])
def test_prefill_scores_of_minus_infinity(gb, cuda, act, kv_len, some):
    minus_infinity(gb, act, kv_len, some, False, 16)


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("cache,value", [("f16", NAN), ("f16", INF), ("q8_0", NAN)])
def test_prefill_tokens_that_see_nothing_stay_zero(gb, cuda, act, cache, value):
    """More tokens than cached rows: the first see nothing, whatever stands in
    the rows that the others see."""
    for which in (0, 1):
        c = R.Cache(gb, CACHE[cache], 2, 64, 16, [12], 3)
        put_value(c, c.pools[which], 0, 1, 1, 20, value)
        check(gb, c, rows(40, 4 * 64, ACT[act], 2), [40], False)


@pytest.mark.parametrize("hd", [64, 128])
def test_prefill_sums_kept_in_the_workspace(gb, cuda, hd):
    """fp32 over enough keys for a running sum, which a row that is computed
    once more leaves to the next one as it should be."""
    c = R.Cache(gb, R.F16, 4, hd, 64, [1100, 300], 3)
    for pos in (1090, 700, 30):
        put_value(c, c.pools[1], 0, pos, 2, 20, INF)
    check(gb, c, rows(400, 4 * hd, F32, 2), [100, 300], False)
