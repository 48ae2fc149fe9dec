// gb_sample.cu -- one token per row of logits: temperature, top-k, top-p,
// min-p, drawn with a given random number.
//
// The weights are integers, w = rint(2^40 e), e = exp((l - max) / T) in fp32,
// so every sum is exact and the token does not depend on how the row is split.
// Every filter keeps a prefix of the order (logit descending, index
// ascending).  With the 64-bit rank (key of the logit, complement of the
// index), unique and ordered the same way, a filter is one cut: kept = rank >=
// cut.
//
// A cluster of SMP_CL CTAs takes a row, each a slice of it in shared memory,
// read from HBM once:
//   maximum      registers, exchanged over the cluster
//   histogram    of (max - l), SMP_BINS linear bins over the distances whose
//                weights are not zero, the rest in the last bin; counts for
//                top-k, weights for top-p
//   cut          each CTA adds up a part of the bins over the cluster; the bin
//                in which the running sum reaches the goal; its tokens go to
//                one CTA, which cuts them by their ranks.  A bin of more than
//                SMP_CAND tokens (many equal logits) is first cut again by the
//                whole cluster.
//   draw         sums by index, the CTA, the warp, the token of the target
#include "gb_common.cuh"
#include "gb_internal.h"
#include "gb_mt.cuh"
#include "gb_paged.cuh"

#include <cooperative_groups.h>

namespace gb {

namespace cg = cooperative_groups;

constexpr int SMP_THREADS = 512;
constexpr int SMP_CL = 8;               // CTAs of a row
constexpr int SMP_BINS = 2048;
constexpr int SMP_CAND = 512;           // tokens of a bin that are ranked directly
constexpr int SMP_W = SMP_THREADS / 32;
static_assert(SMP_CAND <= SMP_THREADS && SMP_BINS % (SMP_CL * 32) == 0, "thread map");
typedef unsigned long long u64;

// Order-preserving key of a logit (NaN and -0 replaced): larger logits have larger keys.
__device__ __forceinline__ uint32_t smp_key(float l) {
    const uint32_t b = __float_as_uint(l);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float smp_logit(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
// NaN is -inf (fmaxf passes over it), -0 is +0.
__device__ __forceinline__ float smp_clean(float l) { return fmaxf(l, -INFINITY) + 0.f; }
// rint(2^40 e), 0 <= e <= 1, as hi 2^23 + lo: hi = rint(2^17 e), lo the rounded
// rest (at most 2^22 in size; e has 24 bits, so the rest is exact).  Rounding
// by adding 2^23 and 1.5 2^23.  Sums of a few thousand parts fit 32 bits.
__device__ __forceinline__ void smp_parts(float e, uint32_t& hi, int& lo) {
    const float y = e * 131072.f, r = y + 8388608.f;
    hi = __float_as_uint(r) - 0x4B000000u;
    const float rest = y - (r - 8388608.f);
    lo = (int)(__float_as_uint(fmaf(rest, 8388608.f, 12582912.f)) - 0x4B400000u);
}
__device__ __forceinline__ u64 smp_join(uint32_t hi, int lo) { return ((u64)hi << 23) + (u64)(long long)lo; }
__device__ __forceinline__ u64 smp_weight(float e) {
    uint32_t hi;
    int lo;
    smp_parts(e, hi, lo);
    return smp_join(hi, lo);
}
// floor(total * part / 2^24), part <= 2^24
__device__ __forceinline__ u64 smp_share(u64 total, uint32_t part) {
    return (total >> 24) * part + (((total & 0xFFFFFFull) * part) >> 24);
}

struct SmpShared {
    uint32_t count[SMP_BINS], wlo[SMP_BINS], whi[SMP_BINS];   // whi:wlo a 64-bit weight
    u64 cand[SMP_CAND], cand_w[SMP_CAND];                     // ranks and weights of a bin's tokens (CTA 0)
    // written by the cluster's CTAs
    u64 peer_max[SMP_CL], peer_a[SMP_CL], peer_b[SMP_CL], peer_sum[SMP_CL];
    u64 cut_a, cut_b, cut_rank, cut_sum;                      // results of a search
    uint32_t cut_bin, n_cand;
    u64 warp64[SMP_W], warp64b[SMP_W];
    u64 tot_a, tot_b;
    uint32_t n_list;
};

// Inclusive sums over the block's threads of two values.
__device__ __forceinline__ void smp_scan2(u64& a, u64& b, u64* sa, u64* sb) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) {
            a += x;
            b += y;
        }
    }
    __syncthreads();
    if (lane == 31) {
        sa[warp] = a;
        sb[warp] = b;
    }
    __syncthreads();
    for (int w = 0; w < warp; w++) {
        a += sa[w];
        b += sb[w];
    }
}

__global__ void __cluster_dims__(SMP_CL, 1, 1) __launch_bounds__(SMP_THREADS, 2)
k_sample(const float* __restrict__ logits, int ldl, int vocab, int slice, const float* __restrict__ temperature,
         const int* __restrict__ top_k, const float* __restrict__ top_p, const float* __restrict__ min_p,
         const float* __restrict__ uu, int* __restrict__ out) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    SmpShared& sh = *reinterpret_cast<SmpShared*>(smem_raw);
    float* x = reinterpret_cast<float*>(smem_raw + (sizeof(SmpShared) + 15) / 16 * 16);   // [slice]
    cg::cluster_group cl = cg::this_cluster();
    const int rank = cl.block_rank(), row = blockIdx.x / SMP_CL;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int i0 = min(rank * slice, vocab), n = min(slice, vocab - i0);   // this CTA's indices i0 .. i0 + n - 1
    const float* src = logits + (size_t)row * ldl + i0;
    griddep_wait();
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");   // every CTA of the cluster runs before remote stores

    // ---- the slice and its maximum; -inf up to whole float4s
    const int n4 = (n + 3) >> 2;
    float mx = -INFINITY;
    if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
#pragma unroll 8
        for (int i = tid; i < n >> 2; i += SMP_THREADS) {
            float4 v = __ldg(reinterpret_cast<const float4*>(src) + i);
            v = make_float4(smp_clean(v.x), smp_clean(v.y), smp_clean(v.z), smp_clean(v.w));
            *reinterpret_cast<float4*>(x + 4 * i) = v;
            mx = fmaxf(mx, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
        }
        const int i = (n & ~3) + tid;
        if (i < 4 * n4) mx = fmaxf(mx, x[i] = i < n ? smp_clean(__ldg(src + i)) : -INFINITY);
    } else {
#pragma unroll 8
        for (int i = tid; i < 4 * n4; i += SMP_THREADS)
            mx = fmaxf(mx, x[i] = i < n ? smp_clean(__ldg(src + i)) : -INFINITY);
    }
    for (int i = tid; i < SMP_BINS; i += SMP_THREADS) sh.count[i] = sh.wlo[i] = sh.whi[i] = 0;
    if (tid == 0) sh.n_cand = 0;
    mx = warp_max(mx);
    if (lane == 0) sh.warp64[warp] = smp_key(mx);
    __syncthreads();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (tid < SMP_CL) {
        u64 b = 0;
#pragma unroll
        for (int w = 0; w < SMP_W; w++) b = sh.warp64[w] > b ? sh.warp64[w] : b;
        cl.map_shared_rank(&sh, tid)->peer_max[rank] = b;
    }
    cl.sync();
    {
        u64 b = 0;
#pragma unroll
        for (int c = 0; c < SMP_CL; c++) b = sh.peer_max[c] > b ? sh.peer_max[c] : b;
        mx = smp_logit((uint32_t)b);
    }
    const float t = temperature ? temperature[row] : 1.f;
    // The first index of the maximum (all CTAs call it).
    auto first_max = [&] {
        uint32_t at = 0xffffffffu;
        for (int i = tid; i < n; i += SMP_THREADS)
            if (x[i] == mx) at = min(at, (uint32_t)(i0 + i));
        at = __reduce_min_sync(0xffffffffu, at);
        __syncthreads();
        if (lane == 0) sh.warp64[warp] = at;
        __syncthreads();
        if (tid < SMP_CL) {
            u64 b = ~0ull;
#pragma unroll
            for (int w = 0; w < SMP_W; w++) b = sh.warp64[w] < b ? sh.warp64[w] : b;
            cl.map_shared_rank(&sh, tid)->peer_max[rank] = b;
        }
        cl.sync();
        u64 b = ~0ull;
#pragma unroll
        for (int c = 0; c < SMP_CL; c++) b = sh.peer_max[c] < b ? sh.peer_max[c] : b;
        return (uint32_t)b;
    };
    if (mx == -INFINITY) {   // nothing to draw
        if (rank == 0 && tid == 0) out[row] = -1;
        return;   // no CTA touches another's memory any more
    }
    if (!(t > 0.f)) {        // greedy
        cl.sync();           // peer_max has been read
        const uint32_t at = first_max();
        if (rank == 0 && tid == 0) out[row] = (int)at;
        return;
    }
    if (mx == INFINITY) {    // certain: the others weigh nothing
        for (int i = tid; i < 4 * n4; i += SMP_THREADS) x[i] = x[i] == INFINITY ? 0.f : -INFINITY;
        mx = 0.f;
        __syncthreads();
    }
    // (l - max) / t correctly rounded: quotient from the rounded reciprocal and
    // one step on its remainder (Markstein, IBM J. Res. Dev. 34, 1990, theorem
    // on division: exact unless t's fraction is all ones), away from over- and
    // underflow; any other t takes the division.  Distances past 30 t weigh
    // nothing: 2^40 e^-30 rounds to 0.
    const float far = -30.f * t, rt = __frcp_rn(t);
    const bool quick = t > 8.6736174e-19f && t < 1.1529215e18f && (__float_as_uint(t) & 0x7fffffu) != 0x7fffffu;
    auto exp_of = [&](float l) {
        const float d = fmaxf(l - mx, far);
        float q;
        if (quick) {
            q = d * rt;
            q = fmaf(fmaf(-t, q, d), rt, q);
        } else {
            q = __fdiv_rn(d, t);
        }
        return expf(q);
    };
    auto weight_of = [&](float l) { return smp_weight(exp_of(l)); };
    const int k = top_k ? top_k[row] : 0;
    const float p = top_p ? top_p[row] : 1.f;
    const float mp = min_p && min_p[row] > 0.f ? fminf(min_p[row], 1.f) : 0.f;
    const bool by_k = k > 0 && k < vocab, by_p = p < 1.f;
    u64 cut = 0;   // kept: rank >= cut

    if (by_k || by_p) {
        // e < 2^-41 rounds to 0 and ln 2^41 = 28.42: the last bin (from 28.47) holds no weight
        const float inv_bin = SMP_BINS / (28.5f * t);
        auto bin_of = [&](float l) {   // monotone in l; 0 where NaN (inf - inf, 0 inf)
            const float d = fminf(fmaxf((mx - l) * inv_bin, 0.f), (float)(SMP_BINS - 1));
            return (int)(__float_as_uint(d + 8388608.f) - 0x4B000000u);   // rounded
        };
        auto rank_of = [&](int i) { return (u64)smp_key(x[i]) << 32 | ~(uint32_t)(i0 + i); };
        auto clear = [&] {
            for (int i = tid; i < SMP_BINS; i += SMP_THREADS) sh.count[i] = sh.wlo[i] = sh.whi[i] = 0;
            __syncthreads();
        };
        auto put = [&](int b, u64 w) {   // a 64-bit sum in two words; the high one rarely moves
            const uint32_t lo = (uint32_t)w, old = atomicAdd(&sh.wlo[b], lo);
            const uint32_t hi = (uint32_t)(w >> 32) + (old + lo < old);
            if (hi) atomicAdd(&sh.whi[b], hi);
        };
        constexpr int PER = SMP_BINS / SMP_CL;
        // The cluster's sums of this thread's bin (a: tokens, b: weights), their
        // running sums over the bins up to it, and the sums of all bins.
        auto merge = [&](u64& own_a, u64& own_b, u64& run_a, u64& run_b, u64& all_a, u64& all_b) {
            cl.sync();   // every histogram is done
            u64 a = 0, b = 0;
            if (tid < PER) {
                const int i = rank * PER + tid;
#pragma unroll
                for (int c = 0; c < SMP_CL; c++) {
                    const SmpShared* o = cl.map_shared_rank(&sh, c);
                    if (by_k) a += o->count[i];
                    if (by_p) b += (u64)o->whi[i] << 32 | o->wlo[i];
                }
            }
            own_a = a;
            own_b = b;
            smp_scan2(a, b, sh.warp64, sh.warp64b);
            if (tid == SMP_THREADS - 1) {
                sh.tot_a = a;
                sh.tot_b = b;
            }
            __syncthreads();
            if (tid < SMP_CL) {
                SmpShared* o = cl.map_shared_rank(&sh, tid);
                o->peer_a[rank] = sh.tot_a;
                o->peer_b[rank] = sh.tot_b;
            }
            cl.sync();
            all_a = all_b = 0;
#pragma unroll
            for (int c = 0; c < SMP_CL; c++) {
                if (c == rank) {
                    a += all_a;
                    b += all_b;
                }
                all_a += sh.peer_a[c];
                all_b += sh.peer_b[c];
            }
            run_a = a;
            run_b = b;
        };
        // The bin at which the running sum reaches goal, and the sums before it: to every CTA.
        auto cross = [&](u64 goal, bool counts, u64 own_a, u64 own_b, u64 run_a, u64 run_b, u64 off_a, u64 off_b) {
            const u64 upto = counts ? off_a + run_a : off_b + run_b, own = counts ? own_a : own_b;
            if (tid < PER && upto - own < goal && goal <= upto)   // one thread of the cluster
                for (int c = 0; c < SMP_CL; c++) {
                    SmpShared* o = cl.map_shared_rank(&sh, c);
                    o->cut_bin = (uint32_t)(rank * PER + tid);
                    o->cut_a = off_a + run_a - own_a;
                    o->cut_b = off_b + run_b - own_b;
                }
            cl.sync();
        };
        // In CTA 0: the candidate at which the sum, from (ga, gb), reaches goal; to every CTA.
        auto resolve = [&](u64 goal, bool counts, u64 ga, u64 gb) {
            const int m = (int)sh.n_cand;
            bool in = tid < m;
            const u64 me = in ? sh.cand[tid] : 0, w = in ? sh.cand_w[tid] : 0;
            int left = m;
            while (left > 32) {   // cut them by their ranks' leading bits, SMP_THREADS bins
                u64 lo = in ? me : ~0ull, hi = me;
                if (!in) hi = 0;
#pragma unroll
                for (int o = 16; o; o >>= 1) {
                    const u64 y = __shfl_xor_sync(0xffffffffu, lo, o), z = __shfl_xor_sync(0xffffffffu, hi, o);
                    lo = y < lo ? y : lo;
                    hi = z > hi ? z : hi;
                }
                __syncthreads();
                if (lane == 0) {
                    sh.warp64[warp] = lo;
                    sh.warp64b[warp] = hi;
                }
                sh.count[tid] = sh.wlo[tid] = sh.whi[tid] = 0;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < SMP_W; i++) {
                    lo = sh.warp64[i] < lo ? sh.warp64[i] : lo;
                    hi = sh.warp64b[i] > hi ? sh.warp64b[i] : hi;
                }
                const int shift = max(0, 64 - __clzll(hi - lo) - 9);   // (hi - lo) >> shift < 512
                const int bin = in ? (int)((hi - me) >> shift) : 0;
                if (in) {
                    atomicAdd(&sh.count[bin], 1u);
                    put(bin, w);
                }
                __syncthreads();
                const u64 own_a = sh.count[tid], own_b = (u64)sh.whi[tid] << 32 | sh.wlo[tid];
                u64 a = own_a, b = own_b;
                smp_scan2(a, b, sh.warp64, sh.warp64b);
                const u64 upto = counts ? ga + a : gb + b, own = counts ? own_a : own_b;
                if (upto - own < goal && goal <= upto) {
                    sh.n_list = (uint32_t)own_a;
                    sh.cut_bin = (uint32_t)tid;
                    sh.tot_a = ga + a - own_a;
                    sh.tot_b = gb + b - own_b;
                }
                __syncthreads();
                ga = sh.tot_a;
                gb = sh.tot_b;
                left = (int)sh.n_list;
                in = in && bin == (int)sh.cut_bin;
            }
            __syncthreads();
            if (tid == 0) sh.n_list = 0;
            __syncthreads();
            if (in) {
                const uint32_t at = atomicAdd(&sh.n_list, 1u);
                sh.cand[at] = me;
                sh.cand_w[at] = w;
            }
            __syncthreads();
            if (warp == 0 && lane < left) {
                const u64 mine = sh.cand[lane], mine_w = sh.cand_w[lane];
                u64 above = ga, above_w = gb;
                for (int j = 0; j < left; j++)
                    if (sh.cand[j] > mine) {
                        above++;
                        above_w += sh.cand_w[j];
                    }
                const u64 before = counts ? above : above_w, own = counts ? 1ull : mine_w;
                if (before < goal && goal <= before + own)
                    for (int c = 0; c < SMP_CL; c++) {
                        SmpShared* o = cl.map_shared_rank(&sh, c);
                        o->cut_rank = mine;
                        o->cut_sum = above_w + mine_w;
                    }
            }
            __syncthreads();
            if (tid == 0) sh.n_cand = 0;
        };

        for (int i = tid; i < n4; i += SMP_THREADS) {
            const float4 v = *reinterpret_cast<const float4*>(x + 4 * i);
            const float l[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int bin = bin_of(l[j]);
                if (by_k) atomicAdd(&sh.count[bin], 1u);
                if (by_p) {
                    const u64 w = weight_of(l[j]);
                    if (w) put(bin, w);
                }
            }
        }
        u64 own_a, own_b, run_a, run_b, all_a, all_b;
        merge(own_a, own_b, run_a, run_b, all_a, all_b);

        // Cut at which the running sum (of tokens or weights) reaches goal, at
        // most the sum of all: its rank, and the weights kept.
        auto search = [&](u64 goal, bool counts, u64& rank_cut, u64& kept) {
            cross(goal, counts, own_a, own_b, run_a, run_b, 0, 0);
            uint32_t bin = sh.cut_bin;
            u64 ga = sh.cut_a, gb = sh.cut_b;
            if (bin == SMP_BINS - 1) return;   // only tokens without weight are cut
            u64 lo = 0, hi = ~0ull;
            int shift = 0;
            for (bool first = true;; first = false) {
                SmpShared* o = cl.map_shared_rank(&sh, 0);
                u64 mn = ~0ull, mxr = 0;
                auto take = [&](int i, float l) {
                    const u64 rk = rank_of(i);
                    mn = rk < mn ? rk : mn;
                    mxr = rk > mxr ? rk : mxr;
                    const uint32_t at = atomicAdd(&o->n_cand, 1u);
                    if (at < SMP_CAND) {
                        o->cand[at] = rk;
                        o->cand_w[at] = weight_of(l);
                    }
                };
                for (int i = tid; i < n4; i += SMP_THREADS) {
                    const float4 v = *reinterpret_cast<const float4*>(x + 4 * i);
                    const float l[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        bool in = bin_of(l[j]) == (int)bin;
                        if (!first) {
                            const u64 rk = rank_of(4 * i + j);
                            in = rk >= lo && rk <= hi && (hi - rk) >> shift == bin;
                        }
                        if (in) take(4 * i + j, l[j]);
                    }
                }
                cl.sync();
                const uint32_t m = o->n_cand;
                if (m <= SMP_CAND) break;
                // too many: bins over the ranks between the first and the last of them
#pragma unroll
                for (int z = 16; z; z >>= 1) {
                    const u64 y = __shfl_xor_sync(0xffffffffu, mn, z), v = __shfl_xor_sync(0xffffffffu, mxr, z);
                    mn = y < mn ? y : mn;
                    mxr = v > mxr ? v : mxr;
                }
                __syncthreads();
                if (lane == 0) {
                    sh.warp64[warp] = mn;
                    sh.warp64b[warp] = mxr;
                }
                __syncthreads();
                if (tid < SMP_CL) {
#pragma unroll
                    for (int i = 0; i < SMP_W; i++) {
                        mn = sh.warp64[i] < mn ? sh.warp64[i] : mn;
                        mxr = sh.warp64b[i] > mxr ? sh.warp64b[i] : mxr;
                    }
                    SmpShared* q = cl.map_shared_rank(&sh, tid);
                    q->peer_a[rank] = mn;
                    q->peer_b[rank] = mxr;
                }
                cl.sync();
                if (rank == 0 && tid == 0) sh.n_cand = 0;
                lo = ~0ull;
                hi = 0;
#pragma unroll
                for (int i = 0; i < SMP_CL; i++) {
                    lo = sh.peer_a[i] < lo ? sh.peer_a[i] : lo;
                    hi = sh.peer_b[i] > hi ? sh.peer_b[i] : hi;
                }
                shift = max(0, 64 - __clzll(hi - lo) - 11);   // (hi - lo) >> shift < 2048
                clear();
                for (int i = tid; i < n; i += SMP_THREADS) {
                    const u64 rk = rank_of(i);
                    if (rk < lo || rk > hi) continue;
                    const int at = (int)((hi - rk) >> shift);
                    if (by_k) atomicAdd(&sh.count[at], 1u);
                    if (by_p) put(at, weight_of(x[i]));
                }
                u64 oa, ob, ra, rb, ta, tb;
                merge(oa, ob, ra, rb, ta, tb);
                cross(goal, counts, oa, ob, ra, rb, ga, gb);
                bin = sh.cut_bin;
                ga = sh.cut_a;
                gb = sh.cut_b;
            }
            if (rank == 0) resolve(goal, counts, ga, gb);
            cl.sync();
            rank_cut = sh.cut_rank;
            kept = sh.cut_sum;
        };
        u64 kept = all_b;
        if (by_k) search((u64)k, true, cut, kept);
        if (by_p) {
            const u64 goal = smp_share(kept, (uint32_t)rintf(fmaxf(p, 0.f) * 16777216.f));
            u64 c2, unused;
            if (goal) search(goal, false, c2, unused);
            else c2 = (u64)smp_key(mx) << 32 | ~first_max();   // the first token alone
            cut = c2 > cut ? c2 : cut;
        }
    }

    // ---- the draw, in index order: warps take consecutive runs of the slice, lanes four neighbours
    const int run = (slice / 4 + SMP_W - 1) / SMP_W;
    const int r0 = min(warp * run, n4), r1 = min(r0 + run, n4);
    const float cut_l = cut ? smp_logit((uint32_t)(cut >> 32)) : -INFINITY;
    const uint32_t cut_i = cut ? ~(uint32_t)cut : 0xffffffffu;   // the last kept index of logit cut_l
    // the weights of float4 i after the filters, as parts
    auto weights = [&](int i, uint32_t (&hi)[4], int (&lo)[4]) {
        const float4 v = i < r1 ? *reinterpret_cast<const float4*>(x + 4 * i)
                                : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        const float l[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            hi[j] = 0;
            lo[j] = 0;
        }
        if (fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) < cut_l) return;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const bool in = l[j] > cut_l || (l[j] == cut_l && (uint32_t)(i0 + 4 * i + j) <= cut_i);
            const float e = exp_of(l[j]);
            uint32_t h;
            int w;
            smp_parts(e, h, w);
            hi[j] = in && e >= mp ? h : 0u;
            lo[j] = in && e >= mp ? w : 0;
        }
    };
    u64 sum = 0;
    {
        uint32_t h4[4], h = 0;   // a lane's part of a slice: at most 2^15 / 512 float4s, 2^17 x 2^8
        int l4[4], l = 0;
        for (int i = r0 + lane; i < r1; i += 32) {
            weights(i, h4, l4);
            h += h4[0] + h4[1] + h4[2] + h4[3];
            l += l4[0] + l4[1] + l4[2] + l4[3];
        }
        sum = smp_join(h, l);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncthreads();
    if (lane == 0) sh.warp64[warp] = sum;
    __syncthreads();
    if (tid < SMP_CL) {
        u64 s = 0;
#pragma unroll
        for (int w = 0; w < SMP_W; w++) s += sh.warp64[w];
        cl.map_shared_rank(&sh, tid)->peer_sum[rank] = s;
    }
    cl.sync();   // after this no CTA touches another's memory
    u64 upto = 0, total = 0;
#pragma unroll
    for (int c = 0; c < SMP_CL; c++) {
        if (c < rank) upto += sh.peer_sum[c];
        total += sh.peer_sum[c];
    }
    for (int w = 0; w < warp; w++) upto += sh.warp64[w];
    const float uf = fminf(fmaxf(uu[row], 0.f), 1.f) * 16777216.f;
    const u64 target = smp_share(total, min((uint32_t)uf, 0xFFFFFFu));
    if (target < upto || target >= upto + sum) return;
    for (int i = r0; i < r1; i += 32) {   // the run that holds the target: find the index
        uint32_t h4[4];
        int l4[4];
        weights(i + lane, h4, l4);
        const u64 own = smp_join(h4[0] + h4[1] + h4[2] + h4[3], l4[0] + l4[1] + l4[2] + l4[3]);
        u64 c = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, c, o);
            if (lane >= o) c += y;
        }
        const uint32_t m = __ballot_sync(0xffffffffu, upto + c > target);
        if (m) {
            if (lane == __ffs(m) - 1) {
                u64 at = upto + c - own;
                int j = 0;
                while (j < 3 && at + smp_join(h4[j], l4[j]) <= target) {
                    at += smp_join(h4[j], l4[j]);
                    j++;
                }
                out[row] = i0 + 4 * (i + lane) + j;
            }
            return;
        }
        upto += __shfl_sync(0xffffffffu, c, 31);
    }
}

}  // namespace gb

extern "C" int gb_sample(const float* logits, int ldl, int rows, int vocab, const float* temperature, const int* top_k,
                         const float* top_p, const float* min_p, const float* u, int* out, void* stream) {
    if (!logits || !u || !out || rows < 0 || vocab <= 0 || ldl < vocab) return GB_EINVAL;
    if (vocab > GB_SAMPLE_MAX_VOCAB) return GB_ELIMIT;
    if (rows == 0) return GB_OK;
    if (rows > 0x7fffffff / gb::SMP_CL) return GB_ELIMIT;
    const int slice = ((vocab + gb::SMP_CL - 1) / gb::SMP_CL + 3) / 4 * 4;
    const size_t smem = (sizeof(gb::SmpShared) + 15) / 16 * 16 + (size_t)slice * sizeof(float);
    constexpr size_t most = (sizeof(gb::SmpShared) + 15) / 16 * 16 + (size_t)GB_SAMPLE_MAX_VOCAB / gb::SMP_CL * sizeof(float);
    static_assert(most <= 227 * 1024, "shared memory");
    if (gb::set_smem_once(reinterpret_cast<const void*>(gb::k_sample), (int)most) != cudaSuccess) return GB_ECUDA;
    return gb::launch_pdl(gb::k_sample, dim3(rows * gb::SMP_CL), gb::SMP_THREADS, (int)smem,
                          static_cast<cudaStream_t>(stream), logits, ldl, vocab, slice, temperature, top_k, top_p, min_p,
                          u, out) == cudaSuccess
               ? GB_OK
               : GB_ECUDA;
}
