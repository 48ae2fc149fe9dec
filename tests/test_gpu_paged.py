"""GPU: the paged KV cache (append with RoPE and quantisation, read) against
its formula bit for bit, and the attention over it against a 64-bit form.

Tolerances (relative L2).  F32 activations: the kernels carry 22 significant
bits of q and of the probabilities and sum in fp32; a score of size ~20 turns
2^-22 into 5e-6 of a probability, errors of different keys are independent:
1e-5.  F16 activations: the output's rounding (2^-11 / sqrt 3 = 2.8e-4), the
probabilities' and, for Q8_0, K's and V's rounding to fp16, each of that size,
scores of size ~3 included: 1.5e-3."""
import pytest
import torch

import paged_ref as R
from helpers import rel_l2

pytestmark = pytest.mark.gpu

F32, F16 = torch.float32, torch.float16
TOL = {F32: 1e-5, F16: 1.5e-3}
ACT = {"f32": F32, "f16": F16}
CACHE = {"f16": R.F16, "q8_0": R.Q8_0}


def cu_of(q_lens):
    return torch.tensor([sum(q_lens[:i]) for i in range(len(q_lens) + 1)], dtype=torch.int32, device="cuda")


def rows_of(n, width, dtype, seed, pad=0, scale=1.0):
    """Rows `pad` elements further apart than they are wide."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    buf = torch.full((n, width + pad), 777.0, dtype=dtype, device="cuda")
    buf[:, :width] = (scale * torch.randn(n, width, generator=g, device="cuda")).to(dtype)
    return buf[:, :width]


# ------------------------------------------------------------------ append and read
@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("cache", ["f16", "q8_0"])
@pytest.mark.parametrize("heads,kv,hd,page,q_lens,past", [
    (4, 4, 64, 16, [1], [0]),
    (32, 8, 128, 32, [1, 1, 1], [31, 32, 700]),
    (7, 1, 64, 64, [5, 0, 130, 1], [0, 9, 60, 15]),
    (10, 2, 128, 16, [33, 16, 15], [1, 0, 17]),
    (28, 4, 128, 256, [300], [300]),
])
def test_append_and_read(gb, cuda, act, cache, heads, kv, hd, page, q_lens, past):
    dt, n = ACT[act], sum(q_lens)
    kv_lens = [a + b for a, b in zip(q_lens, past)]
    c = R.Cache(gb, CACHE[cache], kv, hd, page, kv_lens, 5)
    before = [p.clone() for p in c.pools]
    q, k, v = (rows_of(n, w * hd, dt, 10 + i, pad=8 * i) for i, w in enumerate((heads, kv, kv)))
    cs = torch.empty(max(kv_lens) * hd, dtype=F32, device="cuda")
    gb.rope_table(cs, max(kv_lens), hd)
    one = all(x == 1 for x in q_lens)
    batch = gb.KVBatch(len(q_lens), n, c.len, c.table, None if one else cu_of(q_lens))
    q_out = rows_of(n, heads * hd, dt, 1, pad=16)
    gb.kv_append(c.h, batch, k, v, q=q, q_out=q_out, rope_cs=cs)
    pos = torch.cat([torch.arange(p, p + m, device="cuda") for p, m in zip(past, q_lens)])
    turn = cs.view(-1, hd)[pos]
    assert torch.equal(q_out, R.rope(q.float().unflatten(1, (heads, hd)), turn).flatten(1).to(dt))
    # what the pools should hold now: the old rows, the new ones in their places
    for pool, old, x in zip(c.pools, before, (R.rope(k.float().unflatten(1, (kv, hd)), turn),
                                              v.float().unflatten(1, (kv, hd)))):
        rows, scales = c.parts(old)
        seq = torch.cat([torch.full((m,), s, device="cuda") for s, m in enumerate(q_lens)])
        pg, r = c.table[seq, pos // page].long(), pos % page
        if scales is None:
            rows[pg, :, r] = x.half()
        else:
            rows[pg, :, r], scales[pg, :, r] = R.quantise(x)
        assert torch.equal(pool, old)
    # reading the new tokens, then every row
    ko, vo = rows_of(n, kv * hd, dt, 2, pad=8), rows_of(n, kv * hd, dt, 3)
    gb.kv_read(c.h, batch, ko, vo)
    whole = gb.KVBatch(len(q_lens), sum(kv_lens), c.len, c.table, cu_of(kv_lens))
    ka, va = rows_of(sum(kv_lens), kv * hd, F32, 2), rows_of(sum(kv_lens), kv * hd, F32, 3, pad=4)
    gb.kv_read(c.h, whole, ka, va)
    t0 = w0 = 0
    for s, (m, total) in enumerate(zip(q_lens, kv_lens)):
        for pool, new, every in ((c.pools[0], ko, ka), (c.pools[1], vo, va)):
            x = c.get(pool, s, total).float().flatten(1)
            assert torch.equal(every[w0: w0 + total], x)
            assert torch.equal(new[t0: t0 + m], x[total - m:].to(dt))
        t0, w0 = t0 + m, w0 + total
    assert gb.paged_error() == 0


def test_append_without_rope_in_place_and_odd_values(gb, cuda):
    """No rotation; NaN, infinities, zeros, subnormals and values past fp16's
    range in a Q8_0 cache; q rotated in place."""
    kv, hd = 2, 64
    c = R.Cache(gb, R.Q8_0, kv, hd, 16, [1, 1, 1, 1, 1, 1], 3, fill=False)
    x = torch.zeros(6, kv * hd, device="cuda")
    x[0, 3], x[0, 40] = float("nan"), 2.0
    x[1, 0], x[1, 1] = float("inf"), -1.0
    x[2, 5] = 1e-30
    x[3, :] = torch.linspace(-3e38, 3e38, kv * hd, device="cuda")
    x[4, 70] = -float("inf")
    x[5, :] = torch.linspace(-1e-3, 2e-3, kv * hd, device="cuda")
    batch = gb.KVBatch(6, 6, c.len, c.table)
    gb.kv_append(c.h, batch, x, -x)
    for pool, y in zip(c.pools, (x, -x)):
        rows, scales = c.parts(pool)
        codes, d = R.quantise(y.unflatten(1, (kv, hd)))
        pg = c.table[:6, 0].long()
        assert torch.equal(rows[pg, :, 0], codes) and torch.equal(scales[pg, :, 0], d)
    q = rows_of(6, 3 * hd, F32, 9)
    was, cs = q.clone(), torch.empty(4 * hd, device="cuda")
    gb.rope_table(cs, 4, hd)
    gb.kv_append(c.h, batch, x, x, q=q, q_out=q, rope_cs=cs)
    assert torch.equal(q, R.rope(was.unflatten(1, (3, hd)), cs.view(-1, hd)[:1].expand(6, hd)).flatten(1))


def test_padding_and_recorded_errors(gb, cuda):
    """Tokens past cu_seqlens[n_seq] are left alone; a length past the table, a
    page outside the pool and a position before 0 are recorded and skipped."""
    kv, hd = 2, 64
    c = R.Cache(gb, R.F16, kv, hd, 16, [20, 20, 20], 4)
    c.table[1, 1] = c.n_pages + 1000000
    c.len[2] = 10 ** 6
    before = [p.clone() for p in c.pools]
    k = rows_of(8, kv * hd, F32, 1)
    cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
    batch = gb.KVBatch(3, 8, c.len, c.table, cu)   # 5 padding tokens
    gb.kv_append(c.h, batch, k, k)
    assert gb.paged_error(clear=True) == gb.GB_EPOS and gb.paged_error() == 0
    rows, _ = c.parts(before[0])
    rows[c.table[0, 1].long(), :, 3] = k[0].half().view(kv, hd)
    assert torch.equal(c.pools[0], before[0])
    ko = torch.full((8, kv * hd), 5.0, device="cuda")
    gb.kv_read(c.h, batch, ko, ko.clone())
    assert gb.paged_error(clear=True) == gb.GB_EPOS
    assert torch.equal(ko[0], k[0].half().float()) and not ko[1:3].any() and (ko[3:] == 5).all()
    # attention: the other sequences are as they were, the one without a length gets zeros
    c.k[0], c.v[0] = c.get(c.pools[0], 0, 20), c.get(c.pools[1], 0, 20)
    q, out = rows_of(8, 4 * hd, F32, 2), torch.full((8, 4 * hd), 5.0, device="cuda")
    ws = torch.zeros(gb.paged_workspace_bytes(4, kv, hd, 3), dtype=torch.uint8, device="cuda")
    ref = R.attention(q[:1], c, [1])
    for decode in (False, True):
        out.fill_(5)
        if decode:
            gb.paged_attention_decode(c.h, gb.KVBatch(3, 3, c.len, c.table), q, out, ws)
        else:
            gb.paged_attention_prefill(c.h, batch, q, out, ws)
        assert gb.paged_error(clear=True) == gb.GB_EPOS
        assert rel_l2(out[:1].cpu(), ref.cpu()) <= TOL[F32]
        assert not out[2].any() and (out[3:] == 5).all()


# ------------------------------------------------------------------ attention
def check_attention(gb, act, cache, heads, kv, hd, page, q_lens, kv_lens, decode, seed=1, q_scale=1.5, pad=0, ws=None):
    dt = ACT[act]
    c = R.Cache(gb, CACHE[cache], kv, hd, page, kv_lens, seed)
    n = sum(q_lens)
    q = rows_of(n, heads * hd, dt, seed + 1, pad=pad, scale=q_scale)
    out = rows_of(n, heads * hd, dt, seed + 2, pad=2 * pad)
    if ws is None:
        ws = torch.zeros(gb.paged_workspace_bytes(heads, kv, hd, len(q_lens)), dtype=torch.uint8, device="cuda")
    batch = gb.KVBatch(len(q_lens), n, c.len, c.table, None if decode else cu_of(q_lens))
    f = gb.paged_attention_decode if decode else gb.paged_attention_prefill
    ref = R.attention(q, c, q_lens)
    got = []
    for _ in range(2):   # the workspace is as it was after a call; the sums' order is fixed
        out.fill_(3)
        f(c.h, batch, q, out, ws)
        got.append(out.clone())
    assert torch.equal(got[0], got[1])
    assert torch.isfinite(out).all()
    # each row by itself, against its own size; rows without keys are zeros
    err = (out.double() - ref).norm(dim=1)
    size = ref.norm(dim=1)
    assert not out[size == 0].any()
    some = size > 0
    assert n == 0 or (err[some] <= 3 * TOL[dt] * size[some]).all(), (err[some] / size[some]).max().item()
    assert rel_l2(out.cpu(), ref.cpu()) <= TOL[dt]
    if pad:
        assert (out.as_strided((n, pad), (out.stride(0), 1), out.storage_offset() + heads * hd) == 777).all()
    assert gb.paged_error() == 0


DECODE = [
    # heads, kv, hd, page, kv_lens
    (1, 1, 64, 16, [1]),
    (4, 4, 128, 16, [0, 1, 2, 15, 16, 17]),
    (32, 8, 128, 32, [33, 0, 1000, 128, 127, 129]),
    (32, 4, 64, 16, [300, 5, 64, 1, 2049]),
    (6, 2, 128, 64, [63, 64, 65]),
    (5, 1, 128, 128, [4097]),
    (28, 4, 128, 16, [511, 7]),
    (24, 2, 64, 256, [255, 256, 257]),
    (16, 1, 128, 32, [777, 100]),
    (71, 1, 64, 64, [130, 3]),
    (32, 8, 128, 64, [8193]),
    (8, 1, 128, 64, [20011]),
]


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("cache", ["f16", "q8_0"])
@pytest.mark.parametrize("heads,kv,hd,page,kv_lens", DECODE)
def test_decode(gb, cuda, act, cache, heads, kv, hd, page, kv_lens):
    check_attention(gb, act, cache, heads, kv, hd, page, [1] * len(kv_lens), kv_lens, True, pad=8 if kv == 4 else 0)


@pytest.mark.parametrize("cache", ["f16", "q8_0"])
def test_decode_many_sequences(gb, cuda, cache):
    """More sequences than CTAs, lengths from nothing to a few hundred; the
    same workspace serves a smaller batch after it."""
    lens = [(37 * i * i + 11 * i) % 401 for i in range(400)]
    ws = torch.zeros(gb.paged_workspace_bytes(8, 2, 64, 400), dtype=torch.uint8, device="cuda")
    check_attention(gb, "f32", cache, 8, 2, 64, 16, [1] * 400, lens, True, ws=ws)
    check_attention(gb, "f32", cache, 8, 2, 64, 16, [1] * 3, [1200, 0, 31], True, ws=ws)


@pytest.mark.parametrize("cache", ["f16", "q8_0"])
def test_decode_long_among_short(gb, cuda, cache):
    """Long sequences cut over most CTAs between many short ones, and ending
    where another long one begins."""
    lens = [3] * 90 + [9000, 9100, 40, 8900] + [5] * 90 + [30000]
    check_attention(gb, "f32", cache, 4, 2, 64, 32, [1] * len(lens), lens, True)
    lens = [20000, 20000, 20000]
    check_attention(gb, "f32", cache, 2, 1, 64, 32, [1] * len(lens), lens, True)


PREFILL = [
    # heads, kv, hd, page, q_lens, kv_lens
    (1, 1, 64, 16, [1], [1]),
    (4, 4, 128, 16, [17, 1, 0, 64], [17, 1, 0, 64]),
    (32, 8, 128, 32, [100, 129, 3], [100, 129, 3]),
    (32, 4, 64, 16, [1, 130, 31, 77], [1, 130, 31, 77]),
    (6, 2, 128, 64, [70], [200]),                 # a cached prefix
    (5, 1, 128, 128, [33, 150], [1000, 150]),
    (28, 4, 64, 16, [40, 2], [41, 700]),
    (16, 1, 128, 32, [50], [50]),
    (71, 1, 64, 64, [9], [40]),
    (8, 2, 128, 64, [20, 3, 5], [12, 0, 5]),      # tokens before the cache's first position see nothing
    (8, 8, 128, 64, [513], [513]),
    (2, 2, 64, 256, [700], [700]),
    (8, 1, 128, 16, [16], [9000]),                # few rows, a long axis
    (4, 1, 64, 32, [1, 1, 1], [5000, 1, 64]),
]


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("cache", ["f16", "q8_0"])
@pytest.mark.parametrize("heads,kv,hd,page,q_lens,kv_lens", PREFILL)
def test_prefill(gb, cuda, act, cache, heads, kv, hd, page, q_lens, kv_lens):
    check_attention(gb, act, cache, heads, kv, hd, page, q_lens, kv_lens, False, pad=16 if kv == 2 else 0)


@pytest.mark.parametrize("cache", ["f16", "q8_0"])
def test_prefill_fp32_holds_its_precision_over_a_long_axis(gb, cuda, cache):
    """Enough query blocks that the keys are not split over CTAs: one CTA adds
    up all of a row's 6000 keys."""
    check_attention(gb, "f32", cache, 32, 32, 64, 64, [700], [6000], False)


@pytest.mark.parametrize("hd", [64, 128])
def test_prefill_of_many_blocks(gb, cuda, hd):
    """More CTAs than places for a running sum, each over enough keys to need
    one; up to 32 sequences (longest blocks first, empty ones among them) and more."""
    check_attention(gb, "f32", "f16", 8, 8, hd, 32, [300, 0, 1, 700, 129], [900, 40, 777, 700, 1200], False)
    check_attention(gb, "f32", "q8_0", 8, 8, hd, 16, [40 + s % 3 for s in range(36)], [600 + 7 * s for s in range(36)], False)


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("cache", ["f16", "q8_0"])
@pytest.mark.parametrize("scale", [1e-4, 30.0])
def test_flat_and_peaked_scores(gb, cuda, act, cache, scale):
    """Nearly equal scores, and scores hundreds apart (one key takes all)."""
    if scale > 1 and act == "f16" and cache == "q8_0":
        pytest.skip("K's rounding to fp16 moves scores of this size by more than their gaps")
    check_attention(gb, act, cache, 8, 2, 128, 32, [1, 1], [700, 90], True, q_scale=scale)
    check_attention(gb, act, cache, 8, 2, 128, 32, [130, 20], [300, 20], False, q_scale=scale)


def test_values_of_any_size(gb, cuda):
    """q and cache values far from 1: fp32 activations hold their precision."""
    for kscale, vscale, qscale in ((1e-3, 1e-3, 1e3), (100.0, 1e3, 1e-2), (1e-2, 3e4, 1e4)):
        for cache in (R.F16, R.Q8_0):
            c = R.Cache(gb, cache, 2, 128, 32, [300, 77], 8)
            for s, n in enumerate(c.kv_lens):
                g = torch.Generator(device="cuda").manual_seed(s)
                c.k[s] = c.put(c.pools[0], s, kscale * torch.randn(n, 2, 128, generator=g, device="cuda"))
                c.v[s] = c.put(c.pools[1], s, vscale * torch.rand(n, 2, 128, generator=g, device="cuda"))
            ws = torch.zeros(gb.paged_workspace_bytes(8, 2, 128, 2), dtype=torch.uint8, device="cuda")
            for decode, q_lens in ((True, [1, 1]), (False, [150, 40])):
                q = rows_of(sum(q_lens), 8 * 128, F32, 4, scale=qscale)
                out = torch.empty_like(q)
                batch = gb.KVBatch(2, sum(q_lens), c.len, c.table, None if decode else cu_of(q_lens))
                (gb.paged_attention_decode if decode else gb.paged_attention_prefill)(c.h, batch, q, out, ws)
                # scores grow to |q| |k| ~ 100 for the last set: 2^-22 of that in a probability
                assert rel_l2(out.cpu(), R.attention(q, c, q_lens).cpu()) <= 5e-5, (kscale, vscale, cache, decode)


def test_decode_and_prefill_agree_with_the_per_model_cache(gb, cuda):
    """The same K / V in the fp32 head-major cache (gb_prefill_attention) and in
    F16 pages: the values are fp16 in both, so the results agree to fp32."""
    nh, kv, hd, n = 8, 2, 128, 200
    c = R.Cache(gb, R.F16, kv, hd, 32, [n], 6)
    kc, vc = (x[0].float().transpose(0, 1).contiguous() for x in (c.k, c.v))
    q = rows_of(n, nh * hd, F32, 2)
    a, b = torch.empty_like(q), torch.empty_like(q)
    gb.prefill_attention(q, kc, vc, a, n, 0, nh, kv, hd, n)
    ws = torch.zeros(gb.paged_workspace_bytes(nh, kv, hd, 1), dtype=torch.uint8, device="cuda")
    gb.paged_attention_prefill(c.h, gb.KVBatch(1, n, c.len, c.table, cu_of([n])), q, b, ws)
    assert rel_l2(b.cpu(), a.cpu()) <= 1e-5
    one = torch.empty(1, nh * hd, device="cuda")
    gb.paged_attention_decode(c.h, gb.KVBatch(1, 1, c.len, c.table), q[n - 1:], one, ws)
    assert rel_l2(one.cpu(), a[n - 1:].cpu()) <= 1e-5


def test_another_stream_and_a_graph(gb, cuda):
    """On a side stream, and captured once and replayed as the sequences grow."""
    nh, kv, hd, page = 8, 2, 64, 16
    c = R.Cache(gb, R.Q8_0, kv, hd, page, [40, 9], 7)
    q, k = rows_of(2, nh * hd, F32, 1), rows_of(2, kv * hd, F32, 2)
    out = torch.empty_like(q)
    ws = torch.zeros(gb.paged_workspace_bytes(nh, kv, hd, 2), dtype=torch.uint8, device="cuda")
    batch = gb.KVBatch(2, 2, c.len, c.table)
    gb.paged_attention_decode(c.h, batch, q, out, ws)   # first use outside the capture
    gb.kv_append(c.h, batch, k, k)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        gb.kv_append(c.h, batch, k, k)
        gb.paged_attention_decode(c.h, batch, q, out, ws)
    for lens in ([41, 9], [42, 10], [43, 3]):
        c.len.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        c.kv_lens = lens
        c.k, c.v = ([c.get(p, s, n) for s, n in enumerate(lens)] for p in c.pools)
        assert torch.isfinite(c.k[0]).all()
        assert rel_l2(out.cpu(), R.attention(q, c, [1, 1]).cpu()) <= TOL[F32]
    out.zero_()
    torch.cuda.synchronize()
    gb.paged_attention_decode(c.h, batch, q, out, ws, stream=side.cuda_stream)
    side.synchronize()
    assert rel_l2(out.cpu(), R.attention(q, c, [1, 1]).cpu()) <= TOL[F32]


def test_a_cache_past_32_bit_offsets(gb, cuda):
    """Pages whose byte offset in the pool passes 2^32."""
    kv, hd, page = 8, 128, 256
    nbytes = gb.kv_page_bytes(R.F16, kv, hd, page)
    n_pages = (1 << 32) // nbytes + 20
    c = R.Cache(gb, R.F16, kv, hd, page, [700, 90], 2, spare=n_pages - 4)
    c.table[0, :3] = torch.tensor([n_pages - 1, 2, n_pages - 5], dtype=torch.int32)
    c.table[1, 0] = n_pages - 9
    g = torch.Generator(device="cuda").manual_seed(3)
    for s, n in enumerate(c.kv_lens):
        c.k[s] = c.put(c.pools[0], s, torch.randn(n, kv, hd, generator=g, device="cuda"))
        c.v[s] = c.put(c.pools[1], s, torch.randn(n, kv, hd, generator=g, device="cuda"))
    assert c.n_pages == n_pages
    ws = torch.zeros(gb.paged_workspace_bytes(32, kv, hd, 2), dtype=torch.uint8, device="cuda")
    for decode, q_lens in ((True, [1, 1]), (False, [300, 90])):
        q = rows_of(sum(q_lens), 32 * hd, F16, 4)
        out = torch.empty_like(q)
        batch = gb.KVBatch(2, sum(q_lens), c.len, c.table, None if decode else cu_of(q_lens))
        (gb.paged_attention_decode if decode else gb.paged_attention_prefill)(c.h, batch, q, out, ws)
        assert rel_l2(out.cpu(), R.attention(q, c, q_lens).cpu()) <= TOL[F16]
    k = rows_of(390, kv * hd, F16, 5)
    batch = gb.KVBatch(2, 390, c.len, c.table, cu_of([300, 90]))
    gb.kv_append(c.h, batch, k, k)
    ko, vo = torch.empty_like(k), torch.empty_like(k)
    gb.kv_read(c.h, batch, ko, vo)
    assert torch.equal(ko, k) and torch.equal(vo, k)
    assert gb.paged_error() == 0
