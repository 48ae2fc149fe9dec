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
#include "gb_tc.cuh"

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

// ---------------------------------------------------------------- single tokens
// S = Q K^T and O = P V on mma.sync m16n8k16 (fp16 operands, fp32 sums): the
// 16 rows of the A operand are 8 query heads of one KV head twice, the high
// halves (11 bits) of their values in rows 0-7 and the remainders in rows
// 8-15, so that the padding a group of 8 leaves carries fp32 precision for
// free: the two halves of a C fragment are in one thread and are added.  K
// and V enter exactly: halves as they are, Q8_0 codes as whole numbers in
// fp16, their scales applied to the sums of 32 columns (K) or to the
// probabilities of that column block (V).
//
// Work: a step is 16 keys of one (sequence, KV head, 8 query heads); all
// steps of the batch, in that order, are cut into one equal run per CTA
// whatever the sequences' lengths, and the CTA's warps take its steps in turn.
// Each warp streams its own steps through a ring of cp.async stages and keeps
// its own (m, l, O); they meet once per segment (the steps of one such triple
// in this CTA) in shared memory.  A segment cut by CTA borders leaves a
// partial per CTA; the last of them to arrive joins them in CTA order.
//
// The running maximum m moves only when a score exceeds it by more than
// PD_TAU (log2 units); p = 2^(x - m + PD_LIFT) keeps the fp16 parts of small
// probabilities normal.  Q8_0: p times a scale is brought below 2^14 by a
// power of two, 2^-E, shared by the warp; O is in units of 2^E.
constexpr int PD_W = 4;              // warps
constexpr int PD_MAX_CTAS = 4;       // CTAs per SM the workspace has room for
constexpr int PD_MIN_STEPS = 4;      // fewest steps of a CTA
constexpr int PD_HEADS = 8;          // query heads of a segment
constexpr float PD_TAU = 8.f, PD_LIFT = 6.f;

template <int HD, int DT>
struct PdCfg {
    static constexpr bool Q8 = DT == GB_DT_Q8_0;
    static constexpr int KB = 16 * HD * (Q8 ? 1 : 2);   // bytes of a step's K (or V) rows
    static constexpr int SB = Q8 ? HD : 0;              // and of their scales
    static constexpr int STAGE = 2 * (KB + SB);
    static constexpr int NST = Q8 ? 5 : (HD == 128 ? 3 : 5);
    static constexpr int OP = HD + 4;                   // row pitch of the meeting area (bank spread)
    static constexpr int MEET = PD_W * PD_HEADS * OP * 4 + PD_W * PD_HEADS * 8;
    static constexpr int SMEM = PD_W * NST * STAGE + MEET;
};

__device__ __forceinline__ void pd_cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void pd_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x, y as fp16 pairs: the rounded values and what the rounding left.
__device__ __forceinline__ void pd_split(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 r = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&r);
}
// Bytes {lo, hi} of w (each 128 more than a code) as a pair of halves: placed
// in the mantissa of 1024, 1152 taken off (exact).
__device__ __forceinline__ uint32_t pd_codes(uint32_t w, uint32_t sel) {
    uint32_t b = __byte_perm(w, 0x64646464u, sel);
    __half2 h = __hsub2(*reinterpret_cast<__half2*>(&b), __floats2half2_rn(1152.f, 1152.f));
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ float pd_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A walk over steps: sequence s, segment h of it, step st of nst.
struct PdWalk {
    int s, h, st, nst;
    __device__ __forceinline__ void go(int by, const BatchView& b, int H, unsigned* err) {
        st += by;
        while (st >= nst) {
            st -= nst;
            if (++h == H) {
                h = 0;
                do nst = ++s < b.n_seq ? (seq_len(b, s, err) + 15) >> 4 : 0x7fffffff;   // past the end: no step is taken
                while (nst == 0);
            }
        }
    }
};

// Column of position p (fragment order) of an output row.
template <int HD, int DT>
__device__ __forceinline__ int pd_col(int p) {
    const int n = p >> 3, j = p & 7;   // tile, column in the tile
    return DT == GB_DT_F16 ? (n >> 3) * 64 + 8 * j + (n & 7) : (n >> 2) * 32 + 4 * j + (n & 3);
}

template <typename A, int HD, int DT>
__global__ void __launch_bounds__(PD_W * 32)
k_paged_decode(const PagedView c, const BatchView b, const A* __restrict__ q, int ldq, int group, int n_hg,
               A* __restrict__ out, int ldo, unsigned* __restrict__ tickets, float* __restrict__ part, int min_steps,
               unsigned* err) {
    using C = PdCfg<HD, DT>;
    constexpr int NT = HD / 8;   // output tiles of 8 columns
    constexpr int NB = HD / 32;  // 32-column blocks
    extern __shared__ __align__(16) uint8_t sm[];
    __shared__ unsigned long long s_scan[PD_W];
    __shared__ int s_start[4];
    __shared__ unsigned s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int H = c.n_kv * n_hg, seg_cols = HD;

    // ---- the batch's steps and this CTA's run of them
    const int per = (b.n_seq + PD_W * 32 - 1) / (PD_W * 32);
    const int s_lo = min(tid * per, b.n_seq), s_hi = min(s_lo + per, b.n_seq);
    unsigned long long mine = 0;
    for (int s = s_lo; s < s_hi; s++) mine += (seq_len(b, s, err) + 15) >> 4;
    unsigned long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    unsigned long long T = 0, base = 0;
#pragma unroll
    for (int w = 0; w < PD_W; w++) {
        if (w < warp) base += s_scan[w];
        T += s_scan[w];
    }
    T *= H;
    // sequences without keys: zeros
    for (int s = blockIdx.x; s < b.n_seq; s += gridDim.x)
        if (seq_len(b, s, err) == 0)
            for (int i = tid; i < c.n_kv * group * HD; i += PD_W * 32) out[(size_t)s * ldo + i] = (A)0.f;
    const unsigned long long G = min((unsigned long long)gridDim.x, max(1ull, T / min_steps));
    if (blockIdx.x >= G || T == 0) return;
    const unsigned long long a0 = blockIdx.x * T / G, a1 = (blockIdx.x + 1) * T / G;
    {
        unsigned long long at = (base + incl - mine) * H;   // first step of sequence s_lo
        for (int s = s_lo; s < s_hi; s++) {
            const int n = (seq_len(b, s, err) + 15) >> 4;
            const unsigned long long next = at + (unsigned long long)n * H;
            if (a0 >= at && a0 < next) {
                s_start[0] = s;
                s_start[1] = (int)((a0 - at) / n);
                s_start[2] = (int)((a0 - at) % n);
                s_start[3] = n;
            }
            at = next;
        }
    }
    __syncthreads();
    const int total = (int)(a1 - a0);
    PdWalk seg = {s_start[0], s_start[1], s_start[2], s_start[3]};
    PdWalk iss = seg;
    int iss_i = warp;   // local index of the next step to issue
    iss.go(warp, b, H, err);

    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(sm) + warp * C::NST * C::STAGE;
    const uint8_t* ring_p = sm + warp * C::NST * C::STAGE;
    float* meet = reinterpret_cast<float*>(sm + PD_W * C::NST * C::STAGE);
    float2* meet_ml = reinterpret_cast<float2*>(meet + PD_W * PD_HEADS * C::OP);

    int iss_page = 0;
    auto fetch_page = [&] {
        if (iss_i < total) {
            iss_page = page_of(c, b, iss.s, iss.st << 4, err);
            if (iss_page < 0) iss_page = 0;
        }
    };
    fetch_page();
    auto issue = [&](int slot) {
        if (iss_i < total) {
            const int row = (iss.st << 4) & ((1 << c.shift) - 1);
            const size_t off = (size_t)iss_page * c.page_bytes + (size_t)(iss.h / n_hg) * c.slab;
            const uint32_t dst = ring + slot * C::STAGE;
            if (!C::Q8) {   // every lane copies the 16-byte runs that it will use itself
                const uint8_t* ks = c.k + off + (size_t)(row + g) * HD * 2 + t * 16;
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int j = 0; j < NB; j++)
                        pd_cp16(dst + (i * NB + j) * 512 + lane * 16, ks + i * 8 * HD * 2 + j * 64);
                const uint8_t* vs = c.v + off + (size_t)(row + 2 * t) * HD * 2 + g * 16;
#pragma unroll
                for (int kk = 0; kk < 4; kk++)
#pragma unroll
                    for (int j = 0; j < HD / 64; j++)
                        pd_cp16(dst + C::KB + (kk * (HD / 64) + j) * 512 + lane * 16,
                                vs + ((kk >> 1) * 8 + (kk & 1)) * HD * 2 + j * 128);
            } else {   // rows as they lie, 32-byte units exchanged so that the reads below spread over the banks
                constexpr int CPR = HD / 16;   // 16-byte runs per row
#pragma unroll
                for (int i = 0; i < 16 * CPR / 32; i++) {
                    const int r = (i * 32 + lane) / CPR, ch = (i * 32 + lane) % CPR;
                    const int fk = HD == 128 ? (r & 3) : ((r >> 1) & 1), fv = HD == 128 ? ((r >> 1) & 3) : ((r >> 1) & 1);
                    const size_t src = off + (size_t)(row + r) * HD + ch * 16;
                    pd_cp16(dst + r * HD + ((ch ^ (2 * fk)) * 16), c.k + src);
                    pd_cp16(dst + C::KB + r * HD + ((ch ^ (2 * fv)) * 16), c.v + src);
                }
                if (lane < 2 * (HD / 16)) {   // scales: 16 rows of HD / 32 halves
                    const int ch = lane % (HD / 16);
                    const uint8_t* src = (lane < HD / 16 ? c.k : c.v) + off + ((size_t)HD << c.shift) +
                                         (size_t)row * (HD / 16) + ch * 16;
                    pd_cp16(dst + 2 * C::KB + (lane < HD / 16 ? 0 : C::SB) + ch * 16, src);
                }
            }
            iss_i += PD_W;
            iss.go(PD_W, b, H, err);
            fetch_page();
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < C::NST - 1; i++) issue(i);
    int slot = 0;

    const float scale2 = (1.0f / sqrtf((float)HD)) * 1.4426950408889634f;
    int done = 0;            // local index where the segment starts
    int next = warp;         // local index of this warp's next step
    while (done < total) {
        const int seg_n = min(seg.nst - seg.st, total - done);   // steps of this segment here
        const int kvh = seg.h / n_hg, hg = seg.h % n_hg;
        const int n_heads = min(PD_HEADS, group - hg * PD_HEADS);
        const int len = seq_len(b, seg.s, err);
        float m = -INFINITY, l = 0.f, O[NT][4];
        int E = -40;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) O[n][i] = 0.f;
        if (next < done + seg_n) {
            // ---- q of head g: columns 32 j + 8 t .. + 7, scaled by a power of two and split
            uint32_t qa[2 * NB][4];
            float sc;
            {
                float x[NB][8], mx = 0.f;
                const A* src = q + (size_t)seg.s * ldq + (size_t)(kvh * group + hg * PD_HEADS + g) * HD + 8 * t;
#pragma unroll
                for (int j = 0; j < NB; j++) {
#pragma unroll
                    for (int i = 0; i < 8; i++) x[j][i] = 0.f;
                    if (g < n_heads) act_load8(src + 32 * j, x[j]);
#pragma unroll
                    for (int i = 0; i < 8; i++) mx = fmaxf(mx, fabsf(x[j][i]));
                }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const int e = tc::f16_scale_exp(__float_as_uint(mx));
                const float up = tc::pow2f(e);
                sc = scale2 * tc::pow2f(-e);
#pragma unroll
                for (int j = 0; j < NB; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        pd_split(x[j][2 * i] * up, x[j][2 * i + 1] * up, qa[2 * j + (i >> 1)][2 * (i & 1)],
                                 qa[2 * j + (i >> 1)][2 * (i & 1) + 1]);
            }
            for (; next < done + seg_n; next += PD_W) {
                asm volatile("cp.async.wait_group %0;" ::"n"(C::NST - 2) : "memory");
                __syncwarp();
                issue(slot == 0 ? C::NST - 1 : slot - 1);
                const uint8_t* st = ring_p + slot * C::STAGE;
                slot = slot + 1 == C::NST ? 0 : slot + 1;
                const int k0 = (seg.st + next - done) << 4;
                // ---- scores of keys k0 + 8 i + 2 t, + 1
                float x[4];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    if (!C::Q8) {
                        float sa[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int j = 0; j < NB; j++) {
                            const uint4 kk = *reinterpret_cast<const uint4*>(st + (i * NB + j) * 512 + lane * 16);
                            pd_mma(sa, qa[2 * j], kk.x, kk.y);
                            pd_mma(sa, qa[2 * j + 1], kk.z, kk.w);
                        }
                        x[2 * i] = sa[0] + sa[2];
                        x[2 * i + 1] = sa[1] + sa[3];
                    } else {
                        const int r = 8 * i + g;
                        const int f = HD == 128 ? (r & 3) : ((r >> 1) & 1);
                        x[2 * i] = x[2 * i + 1] = 0.f;
                        __half sk[2][NB];   // scales of keys 8 i + 2 t, + 1
                        const uint8_t* sp = st + 2 * C::KB + (8 * i + 2 * t) * (HD / 16);
                        if (HD == 128) *reinterpret_cast<uint4*>(&sk[0][0]) = *reinterpret_cast<const uint4*>(sp);
                        else *reinterpret_cast<uint2*>(&sk[0][0]) = *reinterpret_cast<const uint2*>(sp);
#pragma unroll
                        for (int j = 0; j < NB; j++) {
                            uint2 w = *reinterpret_cast<const uint2*>(st + r * HD + ((j ^ f) * 32) + 8 * t);
                            w.x ^= 0x80808080u;
                            w.y ^= 0x80808080u;
                            float sa[4] = {0.f, 0.f, 0.f, 0.f};
                            pd_mma(sa, qa[2 * j], pd_codes(w.x, 0x4140), pd_codes(w.x, 0x4342));
                            pd_mma(sa, qa[2 * j + 1], pd_codes(w.y, 0x4140), pd_codes(w.y, 0x4342));
                            x[2 * i] = fmaf(sa[0] + sa[2], __half2float(sk[0][j]), x[2 * i]);
                            x[2 * i + 1] = fmaf(sa[1] + sa[3], __half2float(sk[1][j]), x[2 * i + 1]);
                        }
                    }
                }
                // ---- running softmax (base 2); keys past the sequence weigh nothing
                const int left = len - k0;   // valid keys of the step, at least 1
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int key = (i >> 1) * 8 + 2 * t + (i & 1);
                    x[i] = key < left ? x[i] * sc : -INFINITY;
                    mx = fmaxf(mx, x[i]);
                }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                float alpha = 1.f;
                if (mx > m + PD_TAU || m == -INFINITY) {
                    alpha = pd_ex2(m - mx);
                    if (m == -INFINITY) alpha = 0.f;
                    m = mx;
                }
                float p[4];
                const float ml = m - PD_LIFT;
                l *= alpha;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    p[i] = pd_ex2(x[i] - ml);
                    l += p[i];
                }
                // ---- Q8_0: the V scales of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
                __half sv[4][NB];
                if (C::Q8) {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const uint8_t* sp = st + 2 * C::KB + C::SB + (8 * i + 2 * t) * (HD / 16);
                        if (HD == 128) *reinterpret_cast<uint4*>(&sv[2 * i][0]) = *reinterpret_cast<const uint4*>(sp);
                        else *reinterpret_cast<uint2*>(&sv[2 * i][0]) = *reinterpret_cast<const uint2*>(sp);
                    }
                    if (left < 16) {
#pragma unroll
                        for (int i = 0; i < 4; i++)
#pragma unroll
                            for (int j = 0; j < NB; j++)
                                if ((i >> 1) * 8 + 2 * t + (i & 1) >= left) sv[i][j] = __float2half_rn(0.f);
                    }
                    float top = 0.f;
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int j = 0; j < NB; j++) top = fmaxf(top, __half2float(sv[i][j]));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const int e = (int)(__float_as_uint(top) >> 23) - 126;   // top < 2^e
                    if (e > E) {
                        alpha *= tc::pow2f(max(E - e, -126));
                        E = e;
                    }
                }
                if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int i = 0; i < 4; i++) O[n][i] *= alpha;
                }
                // ---- O += P V
                if (!C::Q8) {
                    uint32_t pa[4];
                    pd_split(p[0], p[1], pa[0], pa[1]);
                    pd_split(p[2], p[3], pa[2], pa[3]);
#pragma unroll
                    for (int j = 0; j < HD / 64; j++) {
                        uint32_t v[4][4];
#pragma unroll
                        for (int kk = 0; kk < 4; kk++) {
                            const uint4 w =
                                *reinterpret_cast<const uint4*>(st + C::KB + (kk * (HD / 64) + j) * 512 + lane * 16);
                            const bool in = (kk >> 1) * 8 + 2 * t + (kk & 1) < left;   // stale rows may hold anything
                            v[kk][0] = in ? w.x : 0u;
                            v[kk][1] = in ? w.y : 0u;
                            v[kk][2] = in ? w.z : 0u;
                            v[kk][3] = in ? w.w : 0u;
                        }
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const uint32_t sel = (e & 1) ? 0x7632 : 0x5410;
                            pd_mma(O[j * 8 + e], pa, __byte_perm(v[0][e >> 1], v[1][e >> 1], sel),
                                   __byte_perm(v[2][e >> 1], v[3][e >> 1], sel));
                        }
                    }
                } else {
                    const float down = tc::pow2f(-E);
#pragma unroll
                    for (int i = 0; i < 4; i++) p[i] *= down;
#pragma unroll
                    for (int j = 0; j < NB; j++) {
                        uint32_t pa[4], w[4];
                        pd_split(p[0] * __half2float(sv[0][j]), p[1] * __half2float(sv[1][j]), pa[0], pa[1]);
                        pd_split(p[2] * __half2float(sv[2][j]), p[3] * __half2float(sv[3][j]), pa[2], pa[3]);
#pragma unroll
                        for (int kk = 0; kk < 4; kk++) {
                            const int r = (kk >> 1) * 8 + 2 * t + (kk & 1);
                            const int f = HD == 128 ? ((r >> 1) & 3) : ((r >> 1) & 1);
                            w[kk] = *reinterpret_cast<const uint32_t*>(st + C::KB + r * HD + ((j ^ f) * 32) + 4 * g) ^
                                    0x80808080u;
                        }
#pragma unroll
                        for (int e2 = 0; e2 < 2; e2++) {   // bytes 2 e2, 2 e2 + 1 of the keys' words
                            const uint32_t lo = __byte_perm(w[0], w[1], e2 ? 0x7362 : 0x5140);
                            const uint32_t hi = __byte_perm(w[2], w[3], e2 ? 0x7362 : 0x5140);
                            pd_mma(O[j * 4 + 2 * e2], pa, pd_codes(lo, 0x4140), pd_codes(hi, 0x4140));
                            pd_mma(O[j * 4 + 2 * e2 + 1], pa, pd_codes(lo, 0x4342), pd_codes(hi, 0x4342));
                        }
                    }
                }
            }
        }
        // ---- the warps meet
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        {
            const float u = C::Q8 ? tc::pow2f(max(E, -126)) : 1.f;
            if (t == 0) meet_ml[warp * PD_HEADS + g] = make_float2(m, l);
            float* row = meet + (warp * PD_HEADS + g) * C::OP + 2 * t;
            if (g < n_heads)
#pragma unroll
                for (int n = 0; n < NT; n++)
                    *reinterpret_cast<float2*>(row + 8 * n) = make_float2((O[n][0] + O[n][2]) * u, (O[n][1] + O[n][3]) * u);
        }
        __syncthreads();
        const unsigned long long gs = a0 + done - seg.st, ge = gs + seg.nst;   // the whole segment's steps
        const bool whole = gs >= a0 && ge <= a1;
        const int slot_out = gs >= a0 ? 1 : 0;
        float* mp = part + ((size_t)blockIdx.x * 2 + slot_out) * (PD_HEADS * (HD + 2));
        const size_t o0 = (size_t)seg.s * ldo + (size_t)(kvh * group + hg * PD_HEADS) * HD;
        for (int i = tid; i < n_heads * seg_cols; i += PD_W * 32) {
            const int h = i / HD, p = i % HD;
            float2 ml[PD_W];
            float M = -INFINITY, L = 0.f, V = 0.f;
#pragma unroll
            for (int w = 0; w < PD_W; w++) {
                ml[w] = meet_ml[w * PD_HEADS + h];
                M = fmaxf(M, ml[w].x);
            }
#pragma unroll
            for (int w = 0; w < PD_W; w++) {
                const float f = ml[w].x == -INFINITY ? 0.f : pd_ex2(ml[w].x - M);
                L = fmaf(ml[w].y, f, L);
                V = fmaf(f == 0.f ? 0.f : meet[(w * PD_HEADS + h) * C::OP + p], f, V);
            }
            if (whole) {
                out[o0 + (size_t)h * HD + pd_col<HD, DT>(p)] = (A)(V / L);
            } else {
                mp[2 * PD_HEADS + i] = V;
                if (p == 0) {
                    mp[2 * h] = M;
                    mp[2 * h + 1] = L;
                }
            }
        }
        if (!whole) {
            // the CTAs of the segment: those that hold its first and last step
            const int c0 = (int)(((gs + 1) * G - 1) / T), c1 = (int)((ge * G - 1) / T);
            __syncthreads();
            if (tid == 0) {
                unsigned prev;
                asm volatile("fence.acq_rel.gpu;\n\tatom.acq_rel.gpu.global.add.u32 %0, [%1], 1;"
                             : "=r"(prev)
                             : "l"(tickets + (size_t)seg.s * H + seg.h)
                             : "memory");
                s_last = prev == (unsigned)(c1 - c0);
            }
            __syncthreads();
            if (s_last) {
                constexpr size_t PS = 2 * PD_HEADS * (HD + 2);   // floats of a CTA's two partials
                for (int i = tid; i < n_heads * seg_cols; i += PD_W * 32) {
                    const int h = i / HD, p = i % HD;
                    float M = -INFINITY, L = 0.f, V = 0.f;
                    for (int cc = c0; cc <= c1; cc++) {
                        const float* pp = part + cc * PS + (cc == c0 ? PD_HEADS * (HD + 2) : 0);
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(pp) + h);
                        const float v = __ldcg(pp + 2 * PD_HEADS + i);
                        const float mn = fmaxf(M, ml.x);
                        const float fa = M == -INFINITY ? 0.f : pd_ex2(M - mn), fb = pd_ex2(ml.x - mn);
                        L = fmaf(L, fa, ml.y * fb);
                        V = fmaf(V, fa, v * fb);
                        M = mn;
                    }
                    out[o0 + (size_t)h * HD + pd_col<HD, DT>(p)] = (A)(V / L);
                }
                if (tid == 0) tickets[(size_t)seg.s * H + seg.h] = 0u;   // every CTA has arrived
            }
        }
        __syncthreads();   // the meeting area is free again
        done += seg_n;
        if (done < total) seg.go(seg_n, b, H, err);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Workspace: the decode CTAs' partials, then one ticket per (sequence, KV
// head, 8 query heads), zero between calls.
constexpr size_t PD_PART_BYTES = (size_t)GB_MAX_SMS * PD_MAX_CTAS * 2 * PD_HEADS * (128 + 2) * 4;

template <typename A, int HD, int DT>
static cudaError_t launch_decode(const PagedView& c, const BatchView& b, const void* q, int ldq, int group, void* out,
                                 int ldo, void* ws, unsigned* err, cudaStream_t st) {
    using C = PdCfg<HD, DT>;
    const void* f = reinterpret_cast<const void*>(k_paged_decode<A, HD, DT>);
    cudaError_t e = set_smem_once(f, C::SMEM);
    if (e != cudaSuccess) return e;
    static const int per_sm = [&] {   // CTAs an SM holds: a property of the build
        int n = 0;
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, f, PD_W * 32, C::SMEM);
        return n < 1 ? 1 : n > PD_MAX_CTAS ? PD_MAX_CTAS : n;
    }();
    const int n_hg = (group + PD_HEADS - 1) / PD_HEADS;
    unsigned* tickets = reinterpret_cast<unsigned*>(static_cast<uint8_t*>(ws) + PD_PART_BYTES);
    k_paged_decode<A, HD, DT><<<sm_count() * per_sm, PD_W * 32, C::SMEM, st>>>(
        c, b, static_cast<const A*>(q), ldq, group, n_hg, static_cast<A*>(out), ldo, tickets, static_cast<float*>(ws),
        PD_MIN_STEPS, err);
    return cudaGetLastError();
}

static int paged_attention(const gb_kv_cache* cache, const gb_kv_batch* batch, int dtype, const void* q, int ldq,
                           int n_heads, void* out, int ldo, void* ws, cudaStream_t st, bool decode) {
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
    const int group = n_heads / c.n_kv;
    if (decode) {
        cudaError_t e = cudaErrorInvalidValue;
#define GB_DECODE(T, A, HD, DT)                                \
    if (dtype == T && hd == HD && cache->dtype == DT)          \
        e = launch_decode<A, HD, DT>(c, b, q, ldq, group, out, ldo, ws, err, st);
        GB_DECODE(GB_DT_F32, float, 128, GB_DT_F16) GB_DECODE(GB_DT_F32, float, 128, GB_DT_Q8_0)
        GB_DECODE(GB_DT_F32, float, 64, GB_DT_F16) GB_DECODE(GB_DT_F32, float, 64, GB_DT_Q8_0)
        GB_DECODE(GB_DT_F16, __half, 128, GB_DT_F16) GB_DECODE(GB_DT_F16, __half, 128, GB_DT_Q8_0)
        GB_DECODE(GB_DT_F16, __half, 64, GB_DT_F16) GB_DECODE(GB_DT_F16, __half, 64, GB_DT_Q8_0)
#undef GB_DECODE
        return e == cudaSuccess ? GB_OK : GB_ECUDA;
    }
    const dim3 grid(b.n_tokens, c.n_kv);
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
    const int group = n_heads / n_kv_heads, n_hg = (group + PD_HEADS - 1) / PD_HEADS;
    return PD_PART_BYTES + ((size_t)n_seq * n_kv_heads * n_hg * sizeof(unsigned) + 15) / 16 * 16;
}

extern "C" int gb_paged_attention_decode(const gb_kv_cache* cache, const gb_kv_batch* batch, int dtype, const void* q,
                                         int ldq, int n_heads, void* out, int ldo, void* ws, void* stream) {
    if (!batch || batch->cu_seqlens) return GB_EINVAL;   // one token per sequence
    return paged_attention(cache, batch, dtype, q, ldq, n_heads, out, ldo, ws, static_cast<cudaStream_t>(stream), true);
}

extern "C" int gb_paged_attention_prefill(const gb_kv_cache* cache, const gb_kv_batch* batch, int dtype, const void* q,
                                          int ldq, int n_heads, void* out, int ldo, void* ws, void* stream) {
    return paged_attention(cache, batch, dtype, q, ldq, n_heads, out, ldo, ws, static_cast<cudaStream_t>(stream), false);
}
