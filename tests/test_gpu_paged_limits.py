"""GPU: lengths, pages, tables and workspaces at their limits: what is out of
range is recorded and skipped, and calls next to it are as they were."""
import pytest
import torch

import paged_ref as R
from helpers import rel_l2

pytestmark = pytest.mark.gpu


def cu_of(q_lens):
    return torch.tensor([sum(q_lens[:i]) for i in range(len(q_lens) + 1)], dtype=torch.int32, device="cuda")


def rows_of(n, width, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(n, width, generator=g, device="cuda").to(dtype)


def workspace(gb, heads, c, n_seq):
    return torch.zeros(gb.paged_workspace_bytes(heads, c.n_kv, c.hd, n_seq), dtype=torch.uint8, device="cuda")


def test_a_length_past_the_part_of_a_table(gb, cuda):
    """A view of some of a wide table's columns: a length past them is recorded,
    although the entries beside the view are pages of the pool."""
    c = R.Cache(gb, R.F16, 2, 64, 16, [64, 40], 5, spare=20)
    wide = torch.zeros(2, 9, dtype=torch.int32, device="cuda")
    wide[:, 2:6] = c.table[:, :4].clamp(min=0)
    part = wide[:, 2:6]
    q, out, ws = rows_of(2, 4 * 64, 1), rows_of(2, 4 * 64, 2), workspace(gb, 4, c, 2)
    k = rows_of(2, 2 * 64, 3)
    for lens, bad in (([64, 40], False), ([65, 40], True)):
        n = torch.tensor(lens, dtype=torch.int32, device="cuda")
        step = gb.KVBatch(2, 2, n, part)
        packed = gb.KVBatch(2, 2, n, part, cu_of([1, 1]))
        c.kv_lens = [0 if x > 64 else x for x in lens]   # counts as empty
        ref = R.attention(q, c, [1, 1]).cpu()
        for attend, b in ((gb.paged_attention_decode, step), (gb.paged_attention_prefill, packed)):
            out.fill_(3)
            attend(c.h, b, q, out, ws)
            assert gb.paged_error(clear=True) == (gb.GB_EPOS if bad else 0)
            assert rel_l2(out.cpu(), ref) <= 1e-5
            assert out[0].any().item() != bad
        before = [p.clone() for p in c.pools]
        if bad:
            gb.kv_append(c.h, gb.KVBatch(1, 1, n, part), k, k)
            assert gb.paged_error(clear=True) == gb.GB_EPOS
            assert all(torch.equal(a, b) for a, b in zip(before, c.pools))


@pytest.mark.parametrize("cache", [R.F16, R.Q8_0])
def test_reading_k_or_v_alone(gb, cuda, cache):
    c = R.Cache(gb, cache, 2, 64, 16, [30, 7], 5)
    b = gb.KVBatch(2, 37, c.len, c.table, cu_of([30, 7]))
    for which in (0, 1):
        x = torch.full((37, 128), 3.0, device="cuda")
        gb.kv_read(c.h, b, *((x, None) if which == 0 else (None, x)))
        assert torch.equal(x, torch.cat([c.get(c.pools[which], s, n) for s, n in ((0, 30), (1, 7))]).float().flatten(1))
    assert gb.paged_error() == 0


def test_a_position_past_the_rotation_table(gb, cuda):
    """Recorded; the token is not written and its q_out row is left as it was."""
    c = R.Cache(gb, R.F16, 2, 64, 16, [20, 33], 5)
    before = [p.clone() for p in c.pools]
    cs = torch.empty(32 * 64, device="cuda")
    gb.rope_table(cs, 32, 64)
    q, k, q_out = rows_of(2, 4 * 64, 1), rows_of(2, 2 * 64, 2), torch.full((2, 4 * 64), 3.0, device="cuda")
    gb.kv_append(c.h, gb.KVBatch(2, 2, c.len, c.table), k, k, q=q, q_out=q_out, rope_cs=cs)
    assert gb.paged_error(clear=True) == gb.GB_EPOS
    turn = cs.view(-1, 64)
    assert torch.equal(q_out[:1], R.rope(q[:1].unflatten(1, (4, 64)), turn[19:20]).flatten(1))
    assert (q_out[1] == 3).all()
    for pool, old, x in zip(c.pools, before, (R.rope(k[:1].unflatten(1, (2, 64)), turn[19:20]), k[:1].unflatten(1, (2, 64)))):
        c.parts(old)[0][c.table[0, 1].long(), :, 3] = x[0].half()
        assert torch.equal(pool, old)


PLACES_AT, PLACES = 192 * 2 * (128 + 2) * 128 * 4, 192   # of running sums in the workspace: behind the sums


def test_a_workspace_without_free_places(gb, cuda):
    """Never zeroed, say: the search for a place ends, is recorded, and places
    that a CTA did not take stay taken."""
    c = R.Cache(gb, R.F16, 32, 64, 32, [700, 900], 5)
    q_lens = [700, 900]
    q = rows_of(sum(q_lens), 32 * 64, 1)
    out = torch.empty_like(q)
    ws = workspace(gb, 32, c, 2)
    places = ws[PLACES_AT: PLACES_AT + 4 * PLACES].view(torch.int32)
    batch = gb.KVBatch(2, sum(q_lens), c.len, c.table, cu_of(q_lens))
    places.fill_(1)
    gb.paged_attention_prefill(c.h, batch, q, out, ws)
    assert gb.paged_error(clear=True) == gb.GB_ETIMEOUT
    assert (places == 1).all()
    places.zero_()
    gb.paged_attention_prefill(c.h, batch, q, out, ws)
    assert gb.paged_error() == 0 and not places.any()
    assert rel_l2(out.cpu(), R.attention(q, c, q_lens).cpu()) <= 1e-5


@pytest.mark.parametrize("cache", [R.F16, R.Q8_0])
@pytest.mark.parametrize("hd", [64, 128])
def test_places_with_the_longest_blocks_first(gb, cuda, cache, hd):
    """Up to 32 sequences, and more CTAs than places for a running sum, each
    over enough keys to need one: 32 heads of one each, two tiles of 128 queries a CTA."""
    q_lens, kv_lens = [300, 0, 1, 700, 129], [900, 40, 777, 700, 1200]
    assert sum(-(-n // 256) for n in q_lens) * 32 > PLACES
    c = R.Cache(gb, cache, 32, hd, 32, kv_lens, 5)
    q = rows_of(sum(q_lens), 32 * hd, 1)
    ref = R.attention(q, c, q_lens).cpu()
    out, ws = torch.empty_like(q), workspace(gb, 32, c, 5)
    batch = gb.KVBatch(5, sum(q_lens), c.len, c.table, cu_of(q_lens))
    got = []
    for _ in range(2):
        gb.paged_attention_prefill(c.h, batch, q, out, ws)
        assert rel_l2(out.cpu(), ref) <= 1e-5
        got.append(out.clone())
    assert torch.equal(*got) and gb.paged_error() == 0
    assert not ws[PLACES_AT: PLACES_AT + 4 * PLACES].any()
    assert ws[:PLACES_AT].any()


@pytest.mark.parametrize("cache", [R.F16, R.Q8_0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_a_table_much_wider_than_the_sequences(gb, cuda, cache, dtype):
    """Few rows and a server's table of 8192 positions: a short prompt's keys
    are not cut into pieces of a tile, which would leave partials; a longer
    prompt's are."""
    for n, pieces in ((200, False), (2000, True)):
        c = R.Cache(gb, cache, 2, 128, 32, [n], 5)
        table = torch.full((1, 256), -7, dtype=torch.int32, device="cuda")
        table[:, : c.table.shape[1]] = c.table
        q = rows_of(40, 8 * 128, 1, dtype)
        out, ws = torch.empty_like(q), workspace(gb, 8, c, 1)
        gb.paged_attention_prefill(c.h, gb.KVBatch(1, 40, c.len, table, cu_of([40])), q, out, ws)
        assert rel_l2(out.float().cpu(), R.attention(q, c, [40]).cpu()) <= (1e-5 if dtype == torch.float32 else 1.5e-3)
        assert gb.paged_error() == 0
        assert ws.any().item() == pieces
