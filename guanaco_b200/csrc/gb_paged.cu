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
#include "gb_tc.cuh"

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
    if (!c || !b || !c->k || !c->v || (b->n_seq > 0 && (!b->kv_len || !b->page_table))) return GB_EINVAL;
    if (c->dtype != GB_DT_F16 && c->dtype != GB_DT_Q8_0) return GB_EINVAL;
    if (c->n_kv_heads <= 0 || c->n_pages <= 0) return GB_EINVAL;
    if (c->head_dim != 64 && c->head_dim != 128) return GB_ESHAPE;
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1))) return GB_ESHAPE;
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) return GB_EINVAL;
    if (b->n_seq < 0 || b->n_tokens < 0 || b->table_stride <= 0) return GB_EINVAL;
    if (b->table_width < 0 || b->table_width > b->table_stride) return GB_EINVAL;
    if (!b->cu_seqlens && b->n_tokens != b->n_seq) return GB_EINVAL;
    const int width = b->table_width ? b->table_width : b->table_stride;
    if ((long long)width * c->page_size > 0x7fffffffLL) return GB_ELIMIT;
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
    bv->cap = width * c->page_size;
    return GB_OK;
}

// ---------------------------------------------------------------- where a token goes
// Token t's place: false for padding; pos < 0 or page < 0: nowhere (recorded).
struct Place {
    int pos, page, row;
};
__device__ __forceinline__ bool place_of(const PagedView& c, const BatchView& b, int t, unsigned* err, Place& o) {
    const int s = t < b.n_tokens ? seq_of(b, t) : -1;
    if (s < 0) return false;
    const int end = b.cu ? __ldg(b.cu + s + 1) : t + 1;
    o.pos = seq_len(b, s, err) - (end - t);
    o.page = -1;
    if (o.pos < 0) {
        atomicExch(err, (unsigned)(-GB_EPOS));
        return true;
    }
    o.page = page_of(c, b, s, o.pos, err);
    o.row = o.pos & ((1 << c.shift) - 1);
    return true;
}

// Both kernels stream: a thread takes 8 columns (4 RoPE pairs, a quarter of a
// Q8_0 block: its maximum by two shuffles) of U heads of one token, looks the
// token's place and rotation up once and has the U heads' loads in flight
// together; neighbouring threads take neighbouring columns.  U = 2 where that
// leaves every SM KV_CTAS CTAs, 1 for a decode batch, whose threads would be
// few.  15,179 prompt tokens (fp32, Q8_0) written and read back: 140 us, 5.8
// TB/s; U = 1 153 us; at most 42 registers a thread (without the bound 156 us);
// CTAs that look a few tokens up for all their threads 155 us (the lookup then
// stands before every load).
constexpr int KV_THREADS = 128, KV_CTAS = 16;

// ---------------------------------------------------------------- append
// 8 values of a Q8_0 block whose largest magnitude is mx: their codes to *to,
// the block's scale returned.  x / d correctly rounded is the product with the
// rounded reciprocal and one step on its remainder (Markstein, IBM J. Res. Dev.
// 34, 1990; d has 11 bits, never a fraction of all ones).  Clamped before
// instead of after; adding 1.5 2^23 rounds to an integer, whose two's
// complement is the low byte (the conversions run at a quarter of the rate).
__device__ __forceinline__ __half quantise8(const float (&x)[8], float mx, uint2* to) {
    const __half d = __float2half_rn(fminf(__fdiv_rn(mx, 127.f), 65504.f));
    const float df = __half2float(d), rd = __frcp_rn(df), lim = 127.f * df;
    uint32_t y[8], w[2];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float v = x[j] == x[j] ? fminf(fmaxf(x[j], -lim), lim) : 0.f;
        const float y0 = v * rd;
        y[j] = __float_as_uint(fmaf(fmaf(-df, y0, v), rd, y0) + 12582912.f);
    }
#pragma unroll
    for (int j = 0; j < 2; j++)
        w[j] = __byte_perm(__byte_perm(y[4 * j], y[4 * j + 1], 0x0040),
                           __byte_perm(y[4 * j + 2], y[4 * j + 3], 0x0040), 0x5410);
    *to = df > 0.f ? make_uint2(w[0], w[1]) : make_uint2(0u, 0u);
    return d;
}

// Heads of a token in the order q, k, v.
template <typename A, int HD, int DT, int U>
__global__ void __launch_bounds__(KV_THREADS, 1536 / KV_THREADS)
k_kv_append(const PagedView c, const BatchView b, const A* __restrict__ q, int ldq, int n_heads, A* __restrict__ q_out,
            int ldqo, const A* __restrict__ k, int ldk, const A* __restrict__ v, int ldv,
            const float* __restrict__ rope, int rope_len, unsigned* err) {
    constexpr int TPH = HD / 8;   // threads per head
    const int heads = n_heads + 2 * c.n_kv, slots = (heads + U - 1) / U;   // head i of a thread: slot + i slots
    const unsigned e = blockIdx.x * KV_THREADS + threadIdx.x, per = (unsigned)(slots * TPH);
    const int t = (int)(e / per), slot = (int)(e % per) / TPH, col = (int)(e % TPH) * 8;
    griddep_wait();
    Place at = {-1, -1, 0};
    if (place_of(c, b, t, err, at) && rope && at.pos >= rope_len) {
        atomicExch(err, (unsigned)(-GB_EPOS));
        at.pos = -1;
    }
    const bool ok = at.pos >= 0;
    float x[U][8], cs[8];
#pragma unroll
    for (int i = 0; i < U; i++) {
        const int head = slot + i * slots;
#pragma unroll
        for (int j = 0; j < 8; j++) x[i][j] = 0.f;
        if (ok && head < heads) {
            const A* src = head < n_heads ? q + (size_t)t * ldq + (size_t)head * HD
                         : head < n_heads + c.n_kv ? k + (size_t)t * ldk + (size_t)(head - n_heads) * HD
                                                   : v + (size_t)t * ldv + (size_t)(head - n_heads - c.n_kv) * HD;
            act_load8(src + col, x[i]);
        }
    }
    if (ok && rope) act_load8(rope + (size_t)at.pos * HD + col, cs);
#pragma unroll
    for (int i = 0; i < U; i++) {
        const int head = slot + i * slots;
        if (ok && rope && head < n_heads + c.n_kv) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float a = x[i][2 * j], bb = x[i][2 * j + 1], co = cs[2 * j], si = cs[2 * j + 1];
                x[i][2 * j] = __fsub_rn(__fmul_rn(a, co), __fmul_rn(bb, si));
                x[i][2 * j + 1] = __fadd_rn(__fmul_rn(a, si), __fmul_rn(bb, co));
            }
        }
        float mx = 0.f;
        if (DT == GB_DT_Q8_0) {   // every lane takes part
#pragma unroll
            for (int j = 0; j < 8; j++) mx = fmaxf(mx, fabsf(x[i][j]));   // NaN passed over
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        }
        if (!ok || head >= heads) continue;
        if (head < n_heads) {
            act_store8(q_out + (size_t)t * ldqo + (size_t)head * HD + col, x[i]);
            continue;
        }
        if (at.page < 0) continue;
        const bool is_v = head >= n_heads + c.n_kv;
        uint8_t* slab = (is_v ? c.v : c.k) + (size_t)at.page * c.page_bytes +
                        (size_t)(head - n_heads - (is_v ? c.n_kv : 0)) * c.slab;
        if (DT == GB_DT_F16) {
            *reinterpret_cast<uint4*>(slab + ((size_t)at.row * HD + col) * 2) = pack_half8(x[i]);
        } else {
            const __half d = quantise8(x[i], mx, reinterpret_cast<uint2*>(slab + (size_t)at.row * HD + col));
            if ((col & 31) == 0)
                reinterpret_cast<__half*>(slab + ((size_t)HD << c.shift))[at.row * (HD / 32) + col / 32] = d;
        }
    }
}

// ---------------------------------------------------------------- read
// Heads of a token in the order k, v.
template <typename A, int HD, int DT, int U>
__global__ void __launch_bounds__(KV_THREADS, 1536 / KV_THREADS)
k_kv_read(const PagedView c, const BatchView b, A* __restrict__ ko, int ldk, A* __restrict__ vo, int ldv,
          unsigned* err) {
    constexpr int TPH = HD / 8;
    const int heads = 2 * c.n_kv, slots = (heads + U - 1) / U;
    const unsigned e = blockIdx.x * KV_THREADS + threadIdx.x, per = (unsigned)(slots * TPH);
    const int t = (int)(e / per), slot = (int)(e % per) / TPH, col = (int)(e % TPH) * 8;
    griddep_wait();
    Place at;
    if (!place_of(c, b, t, err, at)) return;
    uint4 w[U];
    __half d[U];
#pragma unroll
    for (int i = 0; i < U; i++) {
        const int head = slot + i * slots;
        const bool is_v = head >= c.n_kv;
        w[i] = make_uint4(0u, 0u, 0u, 0u);   // a row without a place reads as zeros
        d[i] = __float2half_rn(0.f);
        if (at.page < 0 || head >= heads) continue;
        const uint8_t* slab = (is_v ? c.v : c.k) + (size_t)at.page * c.page_bytes +
                              (size_t)(head - (is_v ? c.n_kv : 0)) * c.slab;
        if (DT == GB_DT_F16) {
            w[i] = ldg4(slab + ((size_t)at.row * HD + col) * 2);
        } else {
            const uint2 y = __ldg(reinterpret_cast<const uint2*>(slab + (size_t)at.row * HD + col));
            w[i].x = y.x;
            w[i].y = y.y;
            d[i] = __ldg(reinterpret_cast<const __half*>(slab + ((size_t)HD << c.shift)) + at.row * (HD / 32) + col / 32);
        }
    }
#pragma unroll
    for (int i = 0; i < U; i++) {
        const int head = slot + i * slots;
        if (head >= heads) continue;
        const bool is_v = head >= c.n_kv;
        A* dst = is_v ? vo : ko;
        if (!dst) continue;
        float x[8];
        if (DT == GB_DT_F16) {
            const uint32_t y[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&y[j]));
                x[2 * j] = f.x;
                x[2 * j + 1] = f.y;
            }
        } else {
            const float df = __half2float(d[i]);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const uint32_t y = (j ? w[i].y : w[i].x) ^ 0x80808080u;   // 128 more than the codes
                x[4 * j] = df * tc::byte_as_float<0>(y, 128.f);
                x[4 * j + 1] = df * tc::byte_as_float<1>(y, 128.f);
                x[4 * j + 2] = df * tc::byte_as_float<2>(y, 128.f);
                x[4 * j + 3] = df * tc::byte_as_float<3>(y, 128.f);
            }
        }
        act_store8(dst + (size_t)t * (is_v ? ldv : ldk) + (size_t)(head - (is_v ? c.n_kv : 0)) * HD + col, x);
    }
}

// CTAs of a call over `heads` heads of every token, u of them a thread; 0: too many.
static unsigned kv_grid(int n_tokens, int heads, int hd, int u) {
    const long long threads = (long long)n_tokens * ((heads + u - 1) / u) * (hd / 8);
    return threads > 0x7fffff00LL ? 0u : (unsigned)((threads + KV_THREADS - 1) / KV_THREADS);
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
    if (b.n_seq == 0 || b.n_tokens == 0) return GB_OK;   // (rows of none may be anywhere)
    const int hd = cache->head_dim;
    const long long kvd = (long long)c.n_kv * hd;
    if (!paged_rows_ok(dtype, k, ldk, kvd) || !paged_rows_ok(dtype, v, ldv, kvd)) return GB_EINVAL;
    if (q) {
        if (n_heads <= 0 || !rope_cs || !paged_rows_ok(dtype, q, ldq, (long long)n_heads * hd) ||
            !paged_rows_ok(dtype, q_out, ldqo, (long long)n_heads * hd))
            return GB_EINVAL;
    } else {
        n_heads = 0;
    }
    if (rope_cs && (rope_len <= 0 || (reinterpret_cast<uintptr_t>(rope_cs) & 15))) return GB_EINVAL;
    unsigned* err = paged_err();
    if (!err) return GB_ECUDA;
    const int heads = n_heads + 2 * c.n_kv;
    const bool many = kv_grid(b.n_tokens, heads, hd, 2) >= (unsigned)(KV_CTAS * sm_count());
    const unsigned grid = kv_grid(b.n_tokens, heads, hd, many ? 2 : 1);
    if (!grid) return GB_ELIMIT;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
#define GB_APPEND(A, HD, DT)                                                                                        \
    e = launch_pdl(many ? k_kv_append<A, HD, DT, 2> : k_kv_append<A, HD, DT, 1>, dim3(grid), KV_THREADS, 0, st, c, b,       \
                   static_cast<const A*>(q), ldq, n_heads, static_cast<A*>(q_out), ldqo, static_cast<const A*>(k),   \
                   ldk, static_cast<const A*>(v), ldv, rope_cs, rope_len, err)
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
    if (b.n_seq == 0 || b.n_tokens == 0) return GB_OK;   // (rows of none may be anywhere)
    const int hd = cache->head_dim;
    const long long kvd = (long long)c.n_kv * hd;
    if ((!k && !v) || (k && !paged_rows_ok(dtype, k, ldk, kvd)) || (v && !paged_rows_ok(dtype, v, ldv, kvd))) return GB_EINVAL;
    unsigned* err = paged_err();
    if (!err) return GB_ECUDA;
    const bool many = kv_grid(b.n_tokens, 2 * c.n_kv, hd, 2) >= (unsigned)(KV_CTAS * sm_count());
    const unsigned grid = kv_grid(b.n_tokens, 2 * c.n_kv, hd, many ? 2 : 1);
    if (!grid) return GB_ELIMIT;
    cudaError_t e;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
#define GB_READ(A, HD, DT) \
    e = launch_pdl(many ? k_kv_read<A, HD, DT, 2> : k_kv_read<A, HD, DT, 1>, dim3(grid), KV_THREADS, 0, st, c, b, \
                   static_cast<A*>(k), ldk, static_cast<A*>(v), ldv, err)
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
