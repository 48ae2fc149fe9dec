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
    int cap;            // table width * page_size: no sequence may be longer
};

inline uint32_t paged_slab(int dtype, int hd, int page) {
    return (uint32_t)(dtype == GB_DT_F16 ? page * hd * 2 : page * (hd + hd / 16));
}

// Host-side checks and conversion shared by the entry points.
int paged_views(const gb_kv_cache* c, const gb_kv_batch* b, PagedView* pv, BatchView* bv);
// Activation rows: 16-byte aligned, at least `width` apart and apart by whole
// 16-byte runs.
inline bool paged_rows_ok(int dtype, const void* p, int ld, long long width) {
    return p && !(reinterpret_cast<uintptr_t>(p) & 15) && ld >= width && ld % (dtype == GB_DT_F16 ? 8 : 4) == 0;
}
// Workspace of the attention entry points: partials (of the prompts' CTAs that
// share a row block, only launched when all of them fit the SMs; or of the
// single tokens' CTAs) or the prompts' running sums; then a ticket per row
// block, which marks a running sum's place as taken where blocks are not
// shared; then two per CTA of the single tokens and one per (sequence, KV head,
// 8 query heads).  Tickets are zero between calls, and never where a call of
// another shape leaves partials.
constexpr size_t PAGED_PART_BYTES = (size_t)GB_MAX_SMS * 2 * (128 + 2) * 128 * sizeof(float);
constexpr size_t PAGED_TICKETS_AT = PAGED_PART_BYTES + GB_MAX_SMS * sizeof(unsigned);
// Packed prompts (gb_paged_prefill.cu).
int paged_prefill(const gb_kv_cache* cache, const PagedView& c, const BatchView& b, int dtype, const void* q, int ldq,
                  int n_heads, void* out, int ldo, void* ws, unsigned* err, cudaStream_t st);
// Tensor map of an F16 pool as {hd halves, page_size rows, slabs} with boxes
// {64, rows, 1}, 128-byte swizzle (gb_matvec.cu, beside the other encoders).
bool paged_encode(void* map128, const void* pool, int hd, int page_size, size_t slabs, int rows);
// Tensor map of a pool for steps of 16 rows of one slab: F16 {64 halves, rows,
// hd / 64, slabs}, box {64, 16, hd / 64, 1}, 128-byte swizzle; Q8_0 codes {hd
// bytes, rows, slabs}, box {hd, 16, 1}, hd-byte swizzle.
bool paged_encode_steps(void* map128, const void* pool, int dtype, int hd, int page_size, size_t slabs);
// Launch that may start while the kernel before it on the stream ends
// (programmatic stream serialization): the kernel executes griddepcontrol.wait
// before it touches global memory.
template <typename F, typename... Args>
cudaError_t launch_pdl(F f, dim3 grid, int threads, int smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, f, args...);
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

// ---------------------------------------------------------------- activations
// 8 consecutive activations as fp32, and back.
__device__ __forceinline__ void act_load8(const float* p, float (&x)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void act_load8(const __half* p, float (&x)[8]) {
    const uint4 r = ldg4(p);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ uint4 pack_half8(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void act_store8(float* p, const float (&x)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void act_store8(__half* p, const float (&x)[8]) {
    *reinterpret_cast<uint4*>(p) = pack_half8(x);
}

}  // namespace gb
