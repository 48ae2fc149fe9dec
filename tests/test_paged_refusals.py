"""CPU: the batched-serving entry points refuse what they do not take before
any device work, and say why."""
import ctypes as C

import pytest

P = 1 << 20   # a 16-byte aligned address that a refused call never reads


def cache(gb, **k):
    a = dict(dtype=2, n_kv_heads=2, head_dim=64, page_size=16, n_pages=4, k=P, v=P)
    a.update(k)
    c = gb.KVCache.__new__(gb.KVCache)
    for n, v in a.items():
        setattr(c, n, v)
    return c


def batch(gb, **k):
    a = dict(n_seq=3, n_tokens=3, cu_seqlens=None, kv_len=P, page_table=P, table_stride=8)
    a.update(k)
    b = gb.KVBatch.__new__(gb.KVBatch)
    for n, v in a.items():
        setattr(b, n, v)
    return b


BAD = [
    (dict(dtype=0), {}, "GB_EINVAL"), (dict(dtype=4), {}, "GB_EINVAL"), (dict(n_kv_heads=0), {}, "GB_EINVAL"),
    (dict(n_pages=0), {}, "GB_EINVAL"), (dict(k=None), {}, "GB_EINVAL"), (dict(v=P + 8), {}, "GB_EINVAL"),
    (dict(head_dim=96), {}, "GB_ESHAPE"), (dict(page_size=8), {}, "GB_ESHAPE"), (dict(page_size=48), {}, "GB_ESHAPE"),
    (dict(page_size=512), {}, "GB_ESHAPE"), ({}, dict(n_seq=-1), "GB_EINVAL"), ({}, dict(n_tokens=-1), "GB_EINVAL"),
    ({}, dict(n_tokens=4), "GB_EINVAL"), ({}, dict(kv_len=None), "GB_EINVAL"), ({}, dict(page_table=None), "GB_EINVAL"),
    ({}, dict(table_stride=0), "GB_EINVAL"), ({}, dict(table_stride=1 << 28), "GB_ELIMIT"),
]


@pytest.mark.parametrize("cc,bb,code", BAD)
def test_cache_and_batch(gb, cc, bb, code):
    L, c0, b0 = gb.lib(), cache(gb, **cc), batch(gb, **bb)
    c, b, want = C.addressof(c0), C.addressof(b0), getattr(gb, code)
    assert L.gb_kv_append(c, b, 0, None, 0, 0, None, 0, P, 128, P, 128, None, 0, None) == want
    assert L.gb_kv_read(c, b, 0, P, 128, P, 128, None) == want
    assert L.gb_paged_attention_decode(c, b, 0, P, 256, 4, P, 256, P, None) == want
    assert L.gb_paged_attention_prefill(c, b, 0, P, 256, 4, P, 256, P, None) == want


def test_rows(gb):
    L, c0, b0 = gb.lib(), cache(gb), batch(gb)
    c, b = C.addressof(c0), C.addressof(b0)
    E = gb.GB_EINVAL

    def append(dt=0, q=None, ldq=0, nh=0, qo=None, ldqo=0, k=P, ldk=128, v=P, ldv=128, cs=None, n=0):
        return L.gb_kv_append(c, b, dt, q, ldq, nh, qo, ldqo, k, ldk, v, ldv, cs, n, None)

    assert append(dt=2) == E and append(k=None) == E and append(v=P + 4) == E and append(ldk=127) == E
    assert append(ldv=130) == E and append(dt=1, ldv=132) == E
    assert append(q=P, ldq=256, nh=4, qo=P, ldqo=256) == E                      # q without a table
    assert append(q=P, ldq=256, nh=4, qo=None, cs=P, n=9) == E
    assert append(q=P, ldq=255, nh=4, qo=P, ldqo=256, cs=P, n=9) == E
    assert append(cs=P, n=0) == E and append(cs=P + 4, n=9) == E
    assert L.gb_kv_read(c, b, 0, None, 0, None, 0, None) == E
    assert L.gb_kv_read(c, b, 0, P, 100, None, 0, None) == E
    for f in (L.gb_paged_attention_decode, L.gb_paged_attention_prefill):
        assert f(c, b, 0, P, 256, 3, P, 256, P, None) == E                      # heads not a multiple
        assert f(c, b, 3, P, 256, 4, P, 256, P, None) == E
        assert f(c, b, 0, P, 200, 4, P, 256, P, None) == E
        assert f(c, b, 0, P, 256, 4, P + 4, 256, P, None) == E
        assert f(c, b, 0, P, 256, 4, P, 256, None, None) == E
        assert f(c, b, 0, P, 256, 4, P, 256, P + 8, None) == E
        assert f(None, b, 0, P, 256, 4, P, 256, P, None) == E
        assert f(c, None, 0, P, 256, 4, P, 256, P, None) == E
    packed = batch(gb, cu_seqlens=P)
    assert L.gb_paged_attention_decode(c, C.addressof(packed), 0, P, 256, 4, P, 256, P, None) == E


def test_limits(gb):
    """Sizes that the kernels' indices do not hold."""
    L, c0, b0 = gb.lib(), cache(gb, n_kv_heads=1), batch(gb)
    c, b = C.addressof(c0), C.addressof(b0)
    assert L.gb_paged_attention_prefill(c, b, 0, P, 129 * 64, 129, P, 129 * 64, P, None) == gb.GB_ELIMIT
    many = batch(gb, n_seq=100, n_tokens=100, table_stride=1 << 26)   # 100 x 2^26 steps of 16 positions
    assert L.gb_paged_attention_decode(c, C.addressof(many), 0, P, 256, 4, P, 256, P, None) == gb.GB_ELIMIT


def test_empty_batches_do_nothing(gb):
    L, c0, b0 = gb.lib(), cache(gb), batch(gb, n_seq=0, n_tokens=0)
    c, b = C.addressof(c0), C.addressof(b0)
    assert L.gb_kv_append(c, b, 0, None, 0, 0, None, 0, P, 128, P, 128, None, 0, None) == 0
    assert L.gb_kv_read(c, b, 0, P, 128, P, 128, None) == 0
    assert L.gb_paged_attention_decode(c, b, 0, P, 256, 4, P, 256, P, None) == 0
    assert L.gb_paged_attention_prefill(c, b, 0, P, 256, 4, P, 256, P, None) == 0
    assert L.gb_sample(P, 10, 0, 10, None, None, None, None, P, P, None) == 0


def test_sizes(gb):
    assert gb.kv_page_bytes(1, 8, 128, 32) == 8 * 32 * 256
    assert gb.kv_page_bytes(2, 8, 128, 32) == 8 * 32 * 136
    assert gb.kv_page_bytes(2, 3, 64, 16) == 3 * 16 * 68
    for a in ((0, 8, 128, 32), (2, 0, 128, 32), (2, 8, 80, 32), (2, 8, 128, 24), (2, 8, 128, 8)):
        assert gb.kv_page_bytes(*a) == 0
    assert gb.paged_workspace_bytes(32, 8, 128, 0) > 0
    for a in ((32, 5, 128, 1), (0, 1, 128, 1), (8, 8, 32, 1), (8, 8, 64, -1)):
        assert gb.paged_workspace_bytes(*a) == 0


def test_sampler(gb):
    L, E = gb.lib(), gb.GB_EINVAL
    assert L.gb_sample(None, 10, 1, 10, None, None, None, None, P, P, None) == E
    assert L.gb_sample(P, 9, 1, 10, None, None, None, None, P, P, None) == E
    assert L.gb_sample(P, 10, -1, 10, None, None, None, None, P, P, None) == E
    assert L.gb_sample(P, 10, 1, 0, None, None, None, None, P, P, None) == E
    assert L.gb_sample(P, 10, 1, 10, None, None, None, None, None, P, None) == E
    assert L.gb_sample(P, 10, 1, 10, None, None, None, None, P, None, None) == E
    assert L.gb_sample(P, 300000, 1, 262145, None, None, None, None, P, P, None) == gb.GB_ELIMIT


def test_python_checks(gb):
    import torch
    z = torch.zeros
    i32 = torch.int32
    with pytest.raises(gb.GBError):
        gb.KVCache(2, 2, 64, 16, 4, z(10, dtype=torch.uint8), z(10, dtype=torch.uint8))
    pool = z(4 * gb.kv_page_bytes(2, 2, 64, 16), dtype=torch.uint8)
    c = gb.KVCache(2, 2, 64, 16, 4, pool, pool.clone())
    for kv_len, table, cu in ((z(3), z(3, 8, dtype=i32), None), (z(2, dtype=i32), z(3, 8, dtype=i32), None),
                              (z(3, dtype=i32), z(2, 8, dtype=i32), None),
                              (z(3, dtype=i32), z(3, 8, dtype=i32), z(3, dtype=i32))):
        with pytest.raises(gb.GBError):
            gb.KVBatch(3, 3, kv_len, table, cu)
    b = gb.KVBatch(3, 3, z(3, dtype=i32), z(3, 8, dtype=i32))
    with pytest.raises(gb.GBError):
        gb.kv_append(c, b, z(3, 128), z(3, 64), stream=0)
    with pytest.raises(gb.GBError):
        gb.kv_append(c, b, z(3, 128), z(3, 128, dtype=torch.float16), stream=0)
    with pytest.raises(gb.GBError):
        gb.kv_append(c, b, z(2, 128), z(2, 128), stream=0)
    with pytest.raises(gb.GBError):
        gb.kv_append(c, b, z(3, 128, dtype=torch.bfloat16), z(3, 128, dtype=torch.bfloat16), stream=0)
    with pytest.raises(gb.GBError):
        gb.paged_attention_decode(c, b, z(3, 256), z(3, 256), z(0), stream=0)
    with pytest.raises(gb.GBError):
        gb.sample(z(2, 9), z(2), z(2), stream=0)
    with pytest.raises(gb.GBError):
        gb.sample(z(2, 9), z(2, dtype=i32), z(1), stream=0)
