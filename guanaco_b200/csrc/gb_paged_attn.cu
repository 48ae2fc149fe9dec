// gb_paged_attn.cu -- attention over the paged KV cache: single new tokens
// (gb_paged_attention_decode) and packed prompts (gb_paged_attention_prefill).
//
//   out[t][h] = sum_p softmax_p(q[t][h] . k[p] / sqrt(hd)) v[p],  p <= position of t
//
// A CTA takes one token and one KV head; its warps take the query heads of
// the group.  A warp walks the keys, the lanes share a row's columns, and the
// running maximum m and sum l of the softmax rescale the output by
// exp(m_old - m).  A token without keys gets zeros.
#include "gb_paged.cuh"

namespace gb {

constexpr int PR_WARPS = 4;

template <typename A, int HD, int DT>
__global__ void __launch_bounds__(PR_WARPS * 32)
k_paged_attn_rows(const PagedView c, const BatchView b, const A* __restrict__ q, int ldq, int group,
                  A* __restrict__ out, int ldo, unsigned* err) {
    constexpr int E = HD / 32;   // columns per lane
    const int t = blockIdx.x, g = blockIdx.y, lane = threadIdx.x & 31;
    const int s = seq_of(b, t);
    if (s < 0) return;
    const int end = b.cu ? __ldg(b.cu + s + 1) : t + 1;
    const int n = seq_len(b, s, err) - (end - t) + 1;   // keys 0 .. n - 1
    const float scale = 1.0f / sqrtf((float)HD);
    for (int j = threadIdx.x >> 5; j < group; j += PR_WARPS) {
        const int h = g * group + j;
        float qv[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
        for (int i = 0; i < E; i++) {
            qv[i] = (float)q[(size_t)t * ldq + (size_t)h * HD + i * 32 + lane];
            o[i] = 0.f;
        }
        for (int p = 0; p < n; p++) {
            const int page = page_of(c, b, s, p, err);
            if (page < 0) continue;
            const int row = p & ((1 << c.shift) - 1);
            const size_t off = (size_t)page * c.page_bytes + (size_t)g * c.slab;
            float d = 0.f, vv[E];
#pragma unroll
            for (int i = 0; i < E; i++) {
                const size_t e = (size_t)row * HD + i * 32 + lane;
                float kk;
                if (DT == GB_DT_F16) {
                    kk = __half2float(reinterpret_cast<const __half*>(c.k + off)[e]);
                    vv[i] = __half2float(reinterpret_cast<const __half*>(c.v + off)[e]);
                } else {
                    const size_t so = off + ((size_t)HD << c.shift) + ((size_t)row * E + i) * 2;
                    kk = __half2float(*reinterpret_cast<const __half*>(c.k + so)) * (float)(int8_t)c.k[off + e];
                    vv[i] = __half2float(*reinterpret_cast<const __half*>(c.v + so)) * (float)(int8_t)c.v[off + e];
                }
                d = fmaf(qv[i], kk, d);
            }
            d = warp_sum(d) * scale;
            const float mn = fmaxf(m, d);
            const float a = expf(m - mn), pr = expf(d - mn);
            l = fmaf(l, a, pr);
            m = mn;
#pragma unroll
            for (int i = 0; i < E; i++) o[i] = fmaf(o[i], a, pr * vv[i]);
        }
        const float inv = l > 0.f ? 1.0f / l : 0.f;
#pragma unroll
        for (int i = 0; i < E; i++)
            out[(size_t)t * ldo + (size_t)h * HD + i * 32 + lane] = (A)(o[i] * inv);
    }
}

static int paged_attention(const gb_kv_cache* cache, const gb_kv_batch* batch, int dtype, const void* q, int ldq,
                           int n_heads, void* out, int ldo, void* ws, cudaStream_t st) {
    PagedView c;
    BatchView b;
    int rc = paged_views(cache, batch, &c, &b);
    if (rc) return rc;
    if (dtype != GB_DT_F32 && dtype != GB_DT_F16) return GB_EINVAL;
    const int hd = cache->head_dim;
    if (n_heads <= 0 || n_heads % c.n_kv || !ws || (reinterpret_cast<uintptr_t>(ws) & 15) || !paged_rows_ok(dtype, q, ldq, n_heads * hd) ||
        !paged_rows_ok(dtype, out, ldo, n_heads * hd))
        return GB_EINVAL;
    if (b.n_tokens == 0) return GB_OK;
    unsigned* err = paged_err();
    if (!err) return GB_ECUDA;
    const dim3 grid(b.n_tokens, c.n_kv);
    const int group = n_heads / c.n_kv;
#define GB_ROWS(A, HD, DT)                                                                                       \
    k_paged_attn_rows<A, HD, DT><<<grid, PR_WARPS * 32, 0, st>>>(c, b, static_cast<const A*>(q), ldq, group,     \
                                                                  static_cast<A*>(out), ldo, err)
#define GB_ROWS_DT(A, HD) \
    if (cache->dtype == GB_DT_F16) GB_ROWS(A, HD, GB_DT_F16); else GB_ROWS(A, HD, GB_DT_Q8_0)
    if (dtype == GB_DT_F32) {
        if (hd == 128) { GB_ROWS_DT(float, 128); } else { GB_ROWS_DT(float, 64); }
    } else {
        if (hd == 128) { GB_ROWS_DT(__half, 128); } else { GB_ROWS_DT(__half, 64); }
    }
#undef GB_ROWS_DT
#undef GB_ROWS
    return cudaGetLastError() == cudaSuccess ? GB_OK : GB_ECUDA;
}

}  // namespace gb

using namespace gb;

extern "C" size_t gb_paged_workspace_bytes(int n_heads, int n_kv_heads, int head_dim, int n_seq) {
    if (n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads || (head_dim != 64 && head_dim != 128) || n_seq < 0)
        return 0;
    return 16;
}

extern "C" int gb_paged_attention_decode(const gb_kv_cache* cache, const gb_kv_batch* batch, int dtype, const void* q,
                                         int ldq, int n_heads, void* out, int ldo, void* ws, void* stream) {
    if (!batch || batch->cu_seqlens) return GB_EINVAL;   // one token per sequence
    return paged_attention(cache, batch, dtype, q, ldq, n_heads, out, ldo, ws, static_cast<cudaStream_t>(stream));
}

extern "C" int gb_paged_attention_prefill(const gb_kv_cache* cache, const gb_kv_batch* batch, int dtype, const void* q,
                                          int ldq, int n_heads, void* out, int ldo, void* ws, void* stream) {
    return paged_attention(cache, batch, dtype, q, ldq, n_heads, out, ldo, ws, static_cast<cudaStream_t>(stream));
}
