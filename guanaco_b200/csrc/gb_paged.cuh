// gb_paged.cuh -- the paged KV cache: how a batch's tokens map to sequences,
// positions, pages and rows, shared by the append, read and attention kernels.
//
// A pool (K and V alike) is n_pages pages; a page is n_kv head slabs; a slab
// holds page_size rows of one KV head:
//   F16   [page_size][hd] halves
//   Q8_0  [page_size][hd] int8 codes, then [page_size][hd / 32] half scales
// The codes of a Q8_0 row are one 16-byte aligned run (GGUF's 34-byte blocks
// would start at every even byte), so rows move in 128-bit accesses.
#pragma once
#include "gb_common.cuh"
#include "gb_internal.h"

namespace gb {

struct PagedView {
    uint8_t *k, *v;
    int n_kv, n_pages;
    int shift;          // log2(page_size)
    uint32_t slab;      // bytes of one (page, KV head)
    size_t page_bytes;  // n_kv * slab
};
struct BatchView {
    const int *cu, *len, *table;
    int n_seq, n_tokens, stride;
    int cap;            // table stride * page_size: no sequence may be longer
};

inline uint32_t paged_slab(int dtype, int hd, int page) {
    return (uint32_t)(dtype == GB_DT_F16 ? page * hd * 2 : page * (hd + hd / 16));
}

// Host-side checks and conversion shared by the entry points.
int paged_views(const gb_kv_cache* c, const gb_kv_batch* b, PagedView* pv, BatchView* bv);
// Activation rows: 16-byte aligned, at least `width` apart and apart by whole
// 16-byte runs.
inline bool paged_rows_ok(int dtype, const void* p, int ld, int width) {
    return p && !(reinterpret_cast<uintptr_t>(p) & 15) && ld >= width && ld % (dtype == GB_DT_F16 ? 8 : 4) == 0;
}
unsigned* paged_err();   // the module's device error word (nullptr: CUDA error)

// Sequence of token t: the largest s with cu[s] <= t (empty sequences share a
// start and are passed over); -1 past the last token.  cu == nullptr: t.
__device__ __forceinline__ int seq_of(const BatchView& b, int t) {
    if (!b.cu) return t < b.n_seq ? t : -1;
    if (t >= __ldg(b.cu + b.n_seq) || t < __ldg(b.cu)) return -1;
    int lo = 0, hi = b.n_seq;   // cu[lo] <= t < cu[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(b.cu + mid) <= t) lo = mid; else hi = mid;
    }
    return lo;
}
// Length of sequence s in the cache; 0 (and GB_EPOS recorded) when it is
// negative or longer than the page table can hold.
__device__ __forceinline__ int seq_len(const BatchView& b, int s, unsigned* err) {
    const int n = __ldg(b.len + s);
    if (n < 0 || n > b.cap) {
        atomicExch(err, (unsigned)(-GB_EPOS));
        return 0;
    }
    return n;
}
// Page of position p of sequence s; -1 (recorded) when the table's entry is
// not a page of the pool.
__device__ __forceinline__ int page_of(const PagedView& c, const BatchView& b, int s, int p, unsigned* err) {
    const int id = __ldg(b.table + (size_t)s * b.stride + (p >> c.shift));
    if ((unsigned)id >= (unsigned)c.n_pages) {
        atomicExch(err, (unsigned)(-GB_EPOS));
        return -1;
    }
    return id;
}

}  // namespace gb
