"""CPU: what the Python layer of the batched-serving entry points refuses
before the library is called, and what it takes."""
import pytest
import torch

i32 = torch.int32


def zeros(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


class Calls:
    """Stands in for the library: records each call's arguments, returns 0."""

    def __init__(self, gb):
        self._gb, self._lib, self.made = gb, gb.lib(), []

    def __getattr__(self, name):
        if name in ("gb_kv_page_bytes", "gb_paged_workspace_bytes"):
            return getattr(self._lib, name)

        def call(*a):
            self.made.append((name, a))
            return 0
        return call


@pytest.fixture
def calls(gb, monkeypatch):
    c = Calls(gb)
    monkeypatch.setattr(gb, "lib", lambda: c)
    return c


def cache(gb, hd=64, kv=2, pages=4, page=16):
    n = pages * gb.kv_page_bytes(gb.DT_Q8_0, kv, hd, page)
    return gb.KVCache(gb.DT_Q8_0, kv, hd, page, pages, zeros(n, dtype=torch.uint8), zeros(n, dtype=torch.uint8))


def batch(gb, n=3, width=8):
    return gb.KVBatch(n, n, zeros(n, dtype=i32), zeros(n, width, dtype=i32))


def test_rotation_tables_that_are_not_rows_of_floats(gb, calls):
    """The kernel reads fp32 rows of head_dim, one after another, rope_len of them."""
    c, b = cache(gb), batch(gb)

    def append(cs):
        gb.kv_append(c, b, zeros(3, 128), zeros(3, 128), rope_cs=cs, stream=0)

    append(zeros(10 * 64))
    append(zeros(10, 32, 2))
    assert [a[13] for _, a in calls.made] == [10, 10]
    for cs in (zeros(10 * 64, dtype=torch.float16), zeros(10, 64, dtype=torch.bfloat16),
               zeros(10, 64, dtype=torch.float64), zeros(10, 128)[:, :64], zeros(64, 10).T, zeros(10 * 64 + 1)):
        with pytest.raises(gb.GBError) as e:
            append(cs)
        assert e.value.rc == gb.GB_EINVAL
    assert len(calls.made) == 2


def test_a_batch_whose_size_is_set_anew(gb, calls):
    """n_seq and n_tokens are fields of the structure: the workspace that a call
    asks for follows them, and no more sequences are taken than the arrays hold."""
    c = cache(gb)
    b = gb.KVBatch(2, 2, zeros(4096, dtype=i32), zeros(4096, 8, dtype=i32))
    small = zeros(gb.paged_workspace_bytes(4, 2, 64, 2), dtype=torch.uint8)
    large = zeros(gb.paged_workspace_bytes(4, 2, 64, 4096), dtype=torch.uint8)
    assert large.numel() > small.numel()
    x = zeros(5000, 256)
    gb.paged_attention_decode(c, b, x, x, small, stream=0)
    b.n_seq = b.n_tokens = 4096
    for attend in (gb.paged_attention_decode, gb.paged_attention_prefill):
        with pytest.raises(gb.GBError) as e:
            attend(c, b, x, x, small, stream=0)
        assert e.value.rc == gb.GB_ESIZE
        attend(c, b, x, x, large, stream=0)
    n = len(calls.made)
    b.n_seq = b.n_tokens = 4097
    kv = zeros(5000, 128)
    for f in (lambda: gb.paged_attention_decode(c, b, x, x, large, stream=0),
              lambda: gb.kv_append(c, b, kv, kv, stream=0), lambda: gb.kv_read(c, b, kv, kv, stream=0)):
        with pytest.raises(gb.GBError):
            f()
    packed = gb.KVBatch(2, 5, zeros(9, dtype=i32), zeros(9, 8, dtype=i32), zeros(4, dtype=i32))
    packed.n_seq = 4   # cu_seqlens holds three
    with pytest.raises(gb.GBError):
        gb.kv_append(c, packed, kv, kv, stream=0)
    assert len(calls.made) == n


def test_a_table_that_is_part_of_a_wider_one(gb, calls):
    """Sequences are bounded by the entries of a row, not by the distance of the
    rows: the last row's entries past them may lie past the end of memory."""
    wide = zeros(3, 16, dtype=i32)
    b = gb.KVBatch(3, 3, zeros(3, dtype=i32), wide[:, 12:])
    assert (b.table_stride, b.table_width) == (16, 4)
    b = gb.KVBatch(3, 3, zeros(3, dtype=i32), wide)
    assert (b.table_stride, b.table_width) == (16, 16)
    with pytest.raises(gb.GBError):
        gb.KVBatch(3, 3, zeros(3, dtype=i32), wide[:, :0])


def test_table_widths(gb):
    import ctypes as C
    P, L = 1 << 20, gb.lib()
    c = gb.KVCache.__new__(gb.KVCache)
    for n, v in dict(dtype=2, n_kv_heads=2, head_dim=64, page_size=16, n_pages=4, k=P, v=P).items():
        setattr(c, n, v)

    def read(stride, width, n=3):
        b = gb.KVBatch.__new__(gb.KVBatch)
        for f, v in dict(n_seq=n, n_tokens=n, kv_len=P, page_table=P, table_stride=stride, table_width=width).items():
            setattr(b, f, v)
        return L.gb_kv_read(C.addressof(c), C.addressof(b), 0, P, 128, P, 128, None)

    assert read(8, -1) == gb.GB_EINVAL and read(8, 9) == gb.GB_EINVAL
    assert read(1 << 28, 1 << 28) == gb.GB_ELIMIT and read(1 << 28, 0) == gb.GB_ELIMIT
    assert read(1 << 28, 8, n=0) == 0 and read(8, 0, n=0) == 0


def test_head_counts_whose_width_passes_32_bits(gb):
    """2^25 heads of 128 are 2^32 columns: no row is that wide."""
    import ctypes as C
    P, L, E = 1 << 20, gb.lib(), gb.GB_EINVAL

    def structs(kv):
        c, b = gb.KVCache.__new__(gb.KVCache), gb.KVBatch.__new__(gb.KVBatch)
        for n, v in dict(dtype=2, n_kv_heads=kv, head_dim=128, page_size=16, n_pages=4, k=P, v=P).items():
            setattr(c, n, v)
        for n, v in dict(n_seq=1, n_tokens=1, kv_len=P, page_table=P, table_stride=8).items():
            setattr(b, n, v)
        return (c, b), C.addressof(c), C.addressof(b)

    keep, c, b = structs(2)
    many = 1 << 25
    assert L.gb_kv_append(c, b, 0, P, 256, many, P, 256, P, 256, P, 256, P, 9, None) == E
    for f in (L.gb_paged_attention_decode, L.gb_paged_attention_prefill):
        assert f(c, b, 0, P, 256, many, P, 256, P, None) == E
    keep, c, b = structs(many)
    assert L.gb_kv_append(c, b, 0, None, 0, 0, None, 0, P, 256, P, 256, None, 0, None) == E
    assert L.gb_kv_read(c, b, 0, P, 256, P, 256, None) == E


def test_strides_past_32_bits_and_gaps(gb, calls):
    """The library's strides are 32-bit, and pools and the workspace are whole
    runs of memory: others are refused, not cut or run over."""
    c, b = cache(gb), batch(gb)
    meta = dict(device="meta")

    def far(rows, width, dtype=torch.float32):   # rows 2^32 + width apart
        return torch.empty(rows, (1 << 32) + width, dtype=dtype, **meta)[:, :width]

    x, kv, ws = zeros(3, 256), zeros(3, 128), zeros(1 << 25, dtype=torch.uint8)
    for f in (lambda: gb.kv_append(c, b, far(3, 128), kv, stream=0), lambda: gb.kv_append(c, b, kv, far(3, 128), stream=0),
              lambda: gb.kv_read(c, b, kv, far(3, 128), stream=0),
              lambda: gb.paged_attention_decode(c, b, far(3, 256), x, ws, stream=0),
              lambda: gb.paged_attention_prefill(c, b, x, far(3, 256), ws, stream=0),
              lambda: gb.sample(far(3, 100), zeros(3, dtype=i32), zeros(3), stream=0),
              lambda: gb.KVBatch(3, 3, zeros(3, dtype=i32), far(3, 8, i32))):
        with pytest.raises(gb.GBError) as e:
            f()
        assert e.value.rc == gb.GB_ELIMIT
    n = 4 * gb.kv_page_bytes(gb.DT_Q8_0, 2, 64, 16)
    whole, gaps = zeros(n, dtype=torch.uint8), zeros(n, 2, dtype=torch.uint8)[:, 0]
    for k, v in ((whole, gaps), (gaps, whole)):
        with pytest.raises(gb.GBError):
            gb.KVCache(gb.DT_Q8_0, 2, 64, 16, 4, k, v)
    with pytest.raises(gb.GBError):
        gb.paged_attention_decode(c, b, x, x, zeros(1 << 25, 2, dtype=torch.uint8)[:, 0], stream=0)
    assert not calls.made


def test_no_tokens_and_no_sequences(gb):
    """Empty tensors have no address: they are taken, and nothing is launched.
    A batch of padding alone (packed tokens, no sequences) too."""
    c = cache(gb)
    z = dict(dtype=i32)
    ws = zeros(gb.paged_workspace_bytes(4, 2, 64, 2), dtype=torch.uint8)
    for n in (0, 3):   # rows
        x, kv = zeros(n, 256), zeros(n, 128)
        batches = [gb.KVBatch(0, n, zeros(0, **z), zeros(0, 8, **z), zeros(1, **z))]
        if n == 0:
            batches += [gb.KVBatch(0, 0, zeros(0, **z), zeros(0, 8, **z)),
                        gb.KVBatch(2, 0, zeros(2, **z), zeros(2, 8, **z), zeros(3, **z))]
        for b in batches:
            gb.kv_append(c, b, kv, kv, q=x, q_out=x, rope_cs=zeros(64), stream=0)
            gb.kv_read(c, b, kv, kv, stream=0)
            gb.paged_attention_prefill(c, b, x, x, ws, stream=0)
            if not b.cu_seqlens:
                gb.paged_attention_decode(c, b, x, x, ws, stream=0)
    gb.sample(zeros(0, 9), zeros(0, **z), zeros(0), stream=0)


def test_one_row_of_any_stride(gb, calls):
    """The distance to the next row of a single one means nothing."""
    def column(width, dtype=torch.float32):
        t = zeros(width, 1, dtype=dtype).t()
        assert t.shape == (1, width) and t.stride() == (1, 1)
        return t

    c = cache(gb)
    b = gb.KVBatch(1, 1, zeros(1, dtype=i32), column(8, i32))
    assert (b.table_stride, b.table_width) == (8, 8)
    gb.kv_append(c, b, column(128), column(128), q=column(256), q_out=column(256), rope_cs=zeros(64), stream=0)
    gb.kv_read(c, b, column(128), column(128), stream=0)
    ws = zeros(gb.paged_workspace_bytes(4, 2, 64, 2), dtype=torch.uint8)
    gb.paged_attention_decode(c, b, column(256), column(256), ws, stream=0)
    gb.sample(column(9), zeros(1, dtype=i32), zeros(1), stream=0)
    ld = {n: [a[i] for i in at] for (n, a), at in zip(calls.made, ((4, 7, 9, 11), (4, 6), (4, 7), (1,)))}
    assert ld == {"gb_kv_append": [256, 256, 128, 128], "gb_kv_read": [128, 128],
                  "gb_paged_attention_decode": [256, 256], "gb_sample": [9]}


def test_reading_k_or_v_alone(gb, calls):
    c, b = cache(gb), batch(gb)
    x = zeros(3, 160)[:, :128]
    gb.kv_read(c, b, x, None, stream=0)
    gb.kv_read(c, b, None, x, stream=0)
    assert [a[3:7] for _, a in calls.made] == [(x.data_ptr(), 160, None, 160), (None, 160, x.data_ptr(), 160)]
    for k, v in ((None, None), (None, zeros(3, 64)), (zeros(2, 128), None)):
        with pytest.raises(gb.GBError):
            gb.kv_read(c, b, k, v, stream=0)
