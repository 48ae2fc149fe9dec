// gb_paged.cu -- writing a paged KV cache (RoPE, quantisation, scatter) and
// reading it back.
//
// Q8_0 of 32 columns: d = half(min(max |x| / 127, 65504)), code = rint(x / d)
// clamped to +-127; d = 0 and NaN give code 0.  The codes are taken against
// the rounded d, so d * code is the nearest value that the stored scale can
// express.  RoPE rounds as the per-model cache's kernels do (a c - b s,
// a s + b c, no contraction).
#include "gb_mt.cuh"
#include "gb_paged.cuh"

#include <atomic>

namespace gb {

__device__ unsigned g_paged_err;

unsigned* paged_err() {
    static std::atomic<unsigned*> at[64];   // per device, looked up once
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
    unsigned* e = at[dev].load(std::memory_order_acquire);
    if (!e) {
        void* p = nullptr;
        if (cudaGetSymbolAddress(&p, g_paged_err) != cudaSuccess) return nullptr;
        e = static_cast<unsigned*>(p);
        at[dev].store(e, std::memory_order_release);
    }
    return e;
}

int paged_views(const gb_kv_cache* c, const gb_kv_batch* b, PagedView* pv, BatchView* bv) {
    if (!c || !b || !c->k || !c->v || !b->kv_len || !b->page_table) return GB_EINVAL;
    if (c->dtype != GB_DT_F16 && c->dtype != GB_DT_Q8_0) return GB_EINVAL;
    if (c->n_kv_heads <= 0 || c->n_pages <= 0) return GB_EINVAL;
    if (c->head_dim != 64 && c->head_dim != 128) return GB_ESHAPE;
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1))) return GB_ESHAPE;
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) return GB_EINVAL;
    if (b->n_seq < 0 || b->n_tokens < 0 || b->table_stride <= 0) return GB_EINVAL;
    if (!b->cu_seqlens && b->n_tokens != b->n_seq) return GB_EINVAL;
    if ((long long)b->table_stride * c->page_size > 0x7fffffffLL) return GB_ELIMIT;
    pv->k = static_cast<uint8_t*>(c->k);
    pv->v = static_cast<uint8_t*>(c->v);
    pv->n_kv = c->n_kv_heads;
    pv->n_pages = c->n_pages;
    pv->shift = __builtin_ctz((unsigned)c->page_size);
    pv->slab = paged_slab(c->dtype, c->head_dim, c->page_size);
    pv->page_bytes = (size_t)pv->slab * c->n_kv_heads;
    bv->cu = b->cu_seqlens;
    bv->len = b->kv_len;
    bv->table = b->page_table;
    bv->n_seq = b->n_seq;
    bv->n_tokens = b->n_tokens;
    bv->stride = b->table_stride;
    bv->cap = b->table_stride * c->page_size;
    return GB_OK;
}

// ---------------------------------------------------------------- append
// A thread takes 8 columns of one head of one token: 4 RoPE pairs, and a
// quarter of a Q8_0 block (its maximum by two shuffles).  Heads of a token in
// the order q, k, v; the threads of a warp take neighbouring columns.
template <typename A, int HD, int DT>
__global__ void __launch_bounds__(256)
k_kv_append(const PagedView c, const BatchView b, const A* __restrict__ q, int ldq, int n_heads, A* __restrict__ q_out,
            int ldqo, const A* __restrict__ k, int ldk, const A* __restrict__ v, int ldv,
            const float* __restrict__ rope, int rope_len, unsigned* err) {
    constexpr int TPH = HD / 8;   // threads per head
    const int per = (n_heads + 2 * c.n_kv) * TPH;
    const unsigned e = blockIdx.x * 256u + threadIdx.x;
    const int t = (int)(e / (unsigned)per), u = (int)(e % (unsigned)per);
    griddep_wait();
    const bool live = t < b.n_tokens;
    int s = -1, pos = -1;
    if (live && (s = seq_of(b, t)) >= 0) {
        const int end = b.cu ? __ldg(b.cu + s + 1) : t + 1;
        const int len = seq_len(b, s, err);
        pos = len - (end - t);
        if (pos < 0) atomicExch(err, (unsigned)(-GB_EPOS));
    }
    int head = u / TPH;
    const int col = (u % TPH) * 8;
    const bool rotate = rope && head < n_heads + c.n_kv;
    if (rotate && pos >= rope_len) {
        atomicExch(err, (unsigned)(-GB_EPOS));
        pos = -1;
    }
    const bool ok = pos >= 0;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (ok) {
        const A* src = head < n_heads ? q + (size_t)t * ldq + (size_t)head * HD
                     : head < n_heads + c.n_kv ? k + (size_t)t * ldk + (size_t)(head - n_heads) * HD
                                               : v + (size_t)t * ldv + (size_t)(head - n_heads - c.n_kv) * HD;
        act_load8(src + col, x);
        if (rotate) {
            float cs[8];
            act_load8(rope + (size_t)pos * HD + col, cs);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float a = x[2 * i], bb = x[2 * i + 1], co = cs[2 * i], si = cs[2 * i + 1];
                x[2 * i] = __fsub_rn(__fmul_rn(a, co), __fmul_rn(bb, si));
                x[2 * i + 1] = __fadd_rn(__fmul_rn(a, si), __fmul_rn(bb, co));
            }
        }
    }
    if (ok && head < n_heads) act_store8(q_out + (size_t)t * ldqo + (size_t)head * HD + col, x);
    // K and V; every lane takes part in the shuffles
    float mx = 0.f;
    if (DT == GB_DT_Q8_0) {
#pragma unroll
        for (int i = 0; i < 8; i++) mx = fmaxf(mx, fabsf(x[i]));   // NaN passed over
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    }
    if (!ok || head < n_heads) return;
    head -= n_heads;
    uint8_t* pool = head < c.n_kv ? c.k : c.v;
    if (head >= c.n_kv) head -= c.n_kv;
    const int page = page_of(c, b, s, pos, err);
    if (page < 0) return;
    const int row = pos & ((1 << c.shift) - 1);
    uint8_t* slab = pool + (size_t)page * c.page_bytes + (size_t)head * c.slab;
    if (DT == GB_DT_F16) {
        *reinterpret_cast<uint4*>(slab + ((size_t)row * HD + col) * 2) = pack_half8(x);
    } else {
        const __half d = __float2half_rn(fminf(__fdiv_rn(mx, 127.f), 65504.f));
        const float df = __half2float(d);
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float y = df > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(x[i], df)), -127.f), 127.f) : 0.f;
            const int code = x[i] == x[i] ? (int)y : 0;
            w[i >> 2] |= (uint32_t)(code & 0xff) << (8 * (i & 3));
        }
        *reinterpret_cast<uint2*>(slab + (size_t)row * HD + col) = make_uint2(w[0], w[1]);
        if ((col & 31) == 0)
            reinterpret_cast<__half*>(slab + ((size_t)HD << c.shift))[row * (HD / 32) + col / 32] = d;
    }
}

// ---------------------------------------------------------------- read
template <typename A, int HD, int DT>
__global__ void __launch_bounds__(256)
k_kv_read(const PagedView c, const BatchView b, A* __restrict__ ko, int ldk, A* __restrict__ vo, int ldv,
          unsigned* err) {
    constexpr int TPH = HD / 8;
    const int per = 2 * c.n_kv * TPH;
    const unsigned e = blockIdx.x * 256u + threadIdx.x;
    const int t = (int)(e / (unsigned)per), u = (int)(e % (unsigned)per);
    griddep_wait();
    if (t >= b.n_tokens) return;
    const int s = seq_of(b, t);
    if (s < 0) return;
    const int end = b.cu ? __ldg(b.cu + s + 1) : t + 1;
    const int pos = seq_len(b, s, err) - (end - t);
    int head = u / TPH;
    const int col = (u % TPH) * 8;
    const bool is_v = head >= c.n_kv;
    if (is_v) head -= c.n_kv;
    if (pos < 0) atomicExch(err, (unsigned)(-GB_EPOS));
    const int page = pos < 0 ? -1 : page_of(c, b, s, pos, err);
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};   // a row without a place reads as zeros
    if (page >= 0) {
        const int row = pos & ((1 << c.shift) - 1);
        const uint8_t* slab = (is_v ? c.v : c.k) + (size_t)page * c.page_bytes + (size_t)head * c.slab;
        if (DT == GB_DT_F16) {
            act_load8(reinterpret_cast<const __half*>(slab) + (size_t)row * HD + col, x);
        } else {
            const uint2 w = __ldg(reinterpret_cast<const uint2*>(slab + (size_t)row * HD + col));
            const float d = __half2float(
                reinterpret_cast<const __half*>(slab + ((size_t)HD << c.shift))[row * (HD / 32) + col / 32]);
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = d * (float)(int8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
        }
    }
    A* dst = is_v ? vo : ko;
    if (dst) act_store8(dst + (size_t)t * (is_v ? ldv : ldk) + (size_t)head * HD + col, x);
}

}  // namespace gb

using namespace gb;

extern "C" size_t gb_kv_page_bytes(int dtype, int n_kv_heads, int head_dim, int page_size) {
    if ((dtype != GB_DT_F16 && dtype != GB_DT_Q8_0) || n_kv_heads <= 0 || (head_dim != 64 && head_dim != 128) ||
        page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
        return 0;
    return (size_t)n_kv_heads * paged_slab(dtype, head_dim, page_size);
}

extern "C" int gb_paged_error(int clear) {
    unsigned v = 0;
    if (cudaMemcpyFromSymbol(&v, gb::g_paged_err, sizeof(v)) != cudaSuccess) return GB_ECUDA;
    if (clear && v) {
        const unsigned z = 0;
        if (cudaMemcpyToSymbol(gb::g_paged_err, &z, sizeof(z)) != cudaSuccess) return GB_ECUDA;
    }
    return -(int)v;
}

extern "C" int gb_kv_append(const gb_kv_cache* cache, const gb_kv_batch* batch, int dtype, const void* q, int ldq,
                            int n_heads, void* q_out, int ldqo, const void* k, int ldk, const void* v, int ldv,
                            const float* rope_cs, int rope_len, void* stream) {
    PagedView c;
    BatchView b;
    int rc = paged_views(cache, batch, &c, &b);
    if (rc) return rc;
    if (dtype != GB_DT_F32 && dtype != GB_DT_F16) return GB_EINVAL;
    const int hd = cache->head_dim, kvd = c.n_kv * hd;
    if (!paged_rows_ok(dtype, k, ldk, kvd) || !paged_rows_ok(dtype, v, ldv, kvd)) return GB_EINVAL;
    if (q) {
        if (n_heads <= 0 || !rope_cs || !paged_rows_ok(dtype, q, ldq, n_heads * hd) ||
            !paged_rows_ok(dtype, q_out, ldqo, n_heads * hd))
            return GB_EINVAL;
    } else {
        n_heads = 0;
    }
    if (rope_cs && (rope_len <= 0 || (reinterpret_cast<uintptr_t>(rope_cs) & 15))) return GB_EINVAL;
    if (b.n_tokens == 0) return GB_OK;
    unsigned* err = paged_err();
    if (!err) return GB_ECUDA;
    const long long threads = (long long)b.n_tokens * (n_heads + 2 * c.n_kv) * (hd / 8);
    if (threads > 0x7fffff00LL) return GB_ELIMIT;
    const unsigned grid = (unsigned)((threads + 255) / 256);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
#define GB_APPEND(A, HD, DT)                                                                                        \
    e = launch_pdl(k_kv_append<A, HD, DT>, dim3(grid), 256, 0, st, c, b, static_cast<const A*>(q), ldq, n_heads,    \
                   static_cast<A*>(q_out), ldqo, static_cast<const A*>(k), ldk, static_cast<const A*>(v), ldv,       \
                   rope_cs, rope_len, err)
#define GB_APPEND_DT(A, HD) \
    if (cache->dtype == GB_DT_F16) GB_APPEND(A, HD, GB_DT_F16); else GB_APPEND(A, HD, GB_DT_Q8_0)
    if (dtype == GB_DT_F32) {
        if (hd == 128) { GB_APPEND_DT(float, 128); } else { GB_APPEND_DT(float, 64); }
    } else {
        if (hd == 128) { GB_APPEND_DT(__half, 128); } else { GB_APPEND_DT(__half, 64); }
    }
#undef GB_APPEND_DT
#undef GB_APPEND
    return e == cudaSuccess ? GB_OK : GB_ECUDA;
}

extern "C" int gb_kv_read(const gb_kv_cache* cache, const gb_kv_batch* batch, int dtype, void* k, int ldk, void* v,
                          int ldv, void* stream) {
    PagedView c;
    BatchView b;
    int rc = paged_views(cache, batch, &c, &b);
    if (rc) return rc;
    if (dtype != GB_DT_F32 && dtype != GB_DT_F16) return GB_EINVAL;
    const int hd = cache->head_dim, kvd = c.n_kv * hd;
    if ((!k && !v) || (k && !paged_rows_ok(dtype, k, ldk, kvd)) || (v && !paged_rows_ok(dtype, v, ldv, kvd))) return GB_EINVAL;
    if (b.n_tokens == 0) return GB_OK;
    unsigned* err = paged_err();
    if (!err) return GB_ECUDA;
    const long long threads = (long long)b.n_tokens * 2 * c.n_kv * (hd / 8);
    if (threads > 0x7fffff00LL) return GB_ELIMIT;
    const unsigned grid = (unsigned)((threads + 255) / 256);
    cudaError_t e;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
#define GB_READ(A, HD, DT) \
    e = launch_pdl(k_kv_read<A, HD, DT>, dim3(grid), 256, 0, st, c, b, static_cast<A*>(k), ldk, static_cast<A*>(v), \
                   ldv, err)
#define GB_READ_DT(A, HD) \
    if (cache->dtype == GB_DT_F16) GB_READ(A, HD, GB_DT_F16); else GB_READ(A, HD, GB_DT_Q8_0)
    if (dtype == GB_DT_F32) {
        if (hd == 128) { GB_READ_DT(float, 128); } else { GB_READ_DT(float, 64); }
    } else {
        if (hd == 128) { GB_READ_DT(__half, 128); } else { GB_READ_DT(__half, 64); }
    }
#undef GB_READ_DT
#undef GB_READ
    return e == cudaSuccess ? GB_OK : GB_ECUDA;
}
