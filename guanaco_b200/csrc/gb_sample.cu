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
//                whole cluster.  A top-k whose bin and those before it hold at
//                most SMP_CAND tokens ends here: CTA 0 filters them and draws,
//                and no other token's weight is computed.
//   draw         sums by index, the CTA, the warp, the token of the target.
//                After a top-p cut each CTA knows its kept weights from its
//                histogram, and only the one with the target goes on.
// A row is a chain of these phases, which the clusters of other rows fill: 1 row
// of 32,000 takes 8.8 us, 256 rows of 128,256 with top-p 225 us = 585 GB/s, 46,000
// cycles a row and cluster: 14,500 until the maximum is known (an HBM round trip
// that each wave of clusters pays), 14,000 for the weights (40 instructions each),
// 17,500 four exchanges over the cluster, the bin's tokens and their ranks.  The
// same rows greedy 71 us, unfiltered or with min-p 120, with top-k 40 129, with
// top-k 2000 194.  Other splits of 256 rows measured
// slower: 16 CTAs a row, three CTAs of 384 threads an SM.
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
    u64 last[32];                                             // the candidates that a search ends with
    u64 cand[SMP_CAND], cand_w[SMP_CAND];                     // ranks of a bin's tokens in this CTA; CTA 0: all, weights
    // written by the cluster's CTAs
    u64 peer_max[SMP_CL], peer_a[SMP_CL], peer_b[SMP_CL], peer_sum[SMP_CL];
    u64 cut_a, cut_rank;                                      // results of a search
    uint32_t cut_bin, cut_n, n_cand, peer_n[SMP_CL];
    u64 warp64[SMP_W], warp64b[SMP_W];
    u64 tot_a;
    uint32_t n_list;
};

// Inclusive sums over the block's threads.
__device__ __forceinline__ u64 smp_scan(u64 a, u64* sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, a, o);
        if (lane >= o) a += x;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = a;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SMP_W; w++) a += w < warp ? sums[w] : 0ull;
    return a;
}

__global__ void __cluster_dims__(SMP_CL, 1, 1) __launch_bounds__(SMP_THREADS, 2)
k_sample(const float* __restrict__ logits, int ldl, int vocab, int slice, const float* __restrict__ temperature,
         const int* __restrict__ top_k, const float* __restrict__ top_p, const float* __restrict__ min_p,
         const float* __restrict__ uu, int* __restrict__ out, bool longest_first) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    SmpShared& sh = *reinterpret_cast<SmpShared*>(smem_raw);
    float* x = reinterpret_cast<float*>(smem_raw + (sizeof(SmpShared) + 15) / 16 * 16);   // [slice]
    cg::cluster_group cl = cg::this_cluster();
    const int rank = cl.block_rank();
    int row = blockIdx.x / SMP_CL;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int i0 = min(rank * slice, vocab), n = min(slice, vocab - i0);   // this CTA's indices i0 .. i0 + n - 1
    griddep_wait();
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");   // every CTA of the cluster runs before remote stores
    if (longest_first) {   // this cluster's row (of at most SMP_THREADS) in the order of their kinds
        const int r = tid;
        const bool in = r < (int)(gridDim.x / SMP_CL);
        int kind = 0;   // a search by weight, the draw alone, a top-k that one CTA ends, greedy
        if (in) {
            const float rt = temperature ? __ldg(temperature + r) : 1.f;
            const int rk = top_k ? __ldg(top_k + r) : 0;
            const bool cut_k = rk > 0 && rk < vocab, cut_p = top_p && __ldg(top_p + r) < 1.f;
            kind = !(rt > 0.f) ? 3 : cut_k && rk <= SMP_CAND ? 2 : !cut_k && !cut_p ? 1 : 0;
        }
        u64 counts = 0, before = 0, all = 0;   // 16 bits a kind
        int at = 0;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const uint32_t m = __ballot_sync(0xffffffffu, in && kind == q);
            counts |= (u64)__popc(m) << (16 * q);
            if (kind == q) at = __popc(m & ((1u << lane) - 1u));
        }
        if (lane == 0) sh.warp64[warp] = counts;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < SMP_W; w++) {
            before += w < warp ? sh.warp64[w] : 0ull;
            all += sh.warp64[w];
        }
        at += (int)(before >> (16 * kind) & 0xffffu);
#pragma unroll
        for (int q = 0; q < 3; q++) at += q < kind ? (int)(all >> (16 * q) & 0xffffu) : 0;
        if (in && at == row) sh.cut_bin = (uint32_t)r;
        __syncthreads();
        row = (int)sh.cut_bin;
    }
    const float* src = logits + (size_t)row * ldl + i0;
    const float t = temperature ? __ldg(temperature + row) : 1.f;
    const int k = top_k ? __ldg(top_k + row) : 0;
    const float p = top_p ? __ldg(top_p + row) : 1.f;
    const float mp = min_p && __ldg(min_p + row) > 0.f ? fminf(__ldg(min_p + row), 1.f) : 0.f;
    const float uf = fminf(fmaxf(__ldg(uu + row), 0.f), 1.f) * 16777216.f;
    for (int i = tid; i < SMP_BINS; i += SMP_THREADS) sh.count[i] = sh.wlo[i] = sh.whi[i] = 0;
    if (tid == 0) sh.n_cand = 0;

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
    mx = warp_max(mx);
    if (lane == 0) sh.warp64[warp] = smp_key(mx);
    __syncthreads();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (warp == 0) {
        const uint32_t b = __reduce_max_sync(0xffffffffu, (uint32_t)sh.warp64[lane % SMP_W]);
        if (lane < SMP_CL) cl.map_shared_rank(&sh, lane)->peer_max[rank] = b;
    }
    cl.sync();
    mx = smp_logit(__reduce_max_sync(0xffffffffu, (uint32_t)sh.peer_max[lane % SMP_CL]));
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
    // underflow; any other t takes the division.  Distances past 28.5 t weigh
    // nothing: 2^40 e^-28.5 rounds to 0.
    const float far = -28.5f * t, rt = __frcp_rn(t);
    const bool quick = t > 8.6736174e-19f && t < 1.1529215e18f && (__float_as_uint(t) & 0x7fffffu) != 0x7fffffu;
    auto exp_of = [&](float l) {
        const float d = fmaxf(l - mx, far);
        float q;
        if (quick) {
            q = d * rt;
            q = fmaf(fmaf(-t, q, d), rt, q);
        } else {
            q = __fdiv_rn(d, fminf(t, 3.4028235e38f));   // (-inf / inf is no number)
        }
        return expf(q);
    };
    auto weight_of = [&](float l) { return smp_weight(exp_of(l)); };
    const bool by_k = k > 0 && k < vocab, by_p = p < 1.f;
    u64 cut = 0;   // kept: rank >= cut
    u64 own_kept = 0;   // this thread's part of this CTA's kept weights, if they are known without a pass
    bool known = false;
    auto block_sum = [&](u64 v) {
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        __syncthreads();
        if (lane == 0) sh.warp64[warp] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int w = 0; w < SMP_W; w++) v += sh.warp64[w];
        return v;
    };

    if (by_k || by_p) {
        // Monotone in l.  The last bin, from 28.493 t on, holds no weight: ln 2^41 = 28.42.
        const float inv_bin = fminf((SMP_BINS - 1) / (28.5f * t), 3.4028235e38f);
        auto bin_of = [&](float l) {   // rounded; no number (t infinite, l masked): the last
            const float d = fmaxf(l - mx, far);
            return (int)min(__float_as_uint(fmaf(d, -inv_bin, 8388608.f)) - 0x4B000000u, (uint32_t)SMP_BINS - 1);
        };
        auto rank_of = [&](int i) { return (u64)smp_key(x[i]) << 32 | ~(uint32_t)(i0 + i); };
        auto clear = [&] {
            for (int i = tid; i < SMP_BINS; i += SMP_THREADS) sh.count[i] = sh.wlo[i] = sh.whi[i] = 0;
            __syncthreads();
        };
        // Weights into bins: a 64-bit sum in two words, the high one moved by a
        // carry or a weight past 2^32 (the few likely tokens).
        auto put = [&](int b, u64 w) {
            const uint32_t lo = (uint32_t)w, old = atomicAdd(&sh.wlo[b], lo);
            const uint32_t hi = (uint32_t)(w >> 32) + (old + lo < old);
            if (hi) atomicAdd(&sh.whi[b], hi);
        };
        constexpr int PER = SMP_BINS / SMP_CL;
        // The cluster's sum of this thread's bin (tokens or weights), the running
        // sum over the bins up to it, and the sum of all bins.
        auto merge = [&](bool counts, u64& own, u64& run, u64& all) {
            cl.sync();   // every histogram is done
            u64 a = 0;
            if (tid < PER) {
                const int i = rank * PER + tid;
#pragma unroll
                for (int c = 0; c < SMP_CL; c++) {
                    const SmpShared* o = cl.map_shared_rank(&sh, c);
                    a += counts ? o->count[i] : (u64)o->whi[i] << 32 | o->wlo[i];
                }
            }
            own = a;
            a = smp_scan(a, sh.warp64);
            if (tid == SMP_THREADS - 1) sh.tot_a = a;
            __syncthreads();
            if (tid < SMP_CL) cl.map_shared_rank(&sh, tid)->peer_a[rank] = sh.tot_a;
            cl.sync();
            all = 0;
#pragma unroll
            for (int c = 0; c < SMP_CL; c++) {
                if (c == rank) a += all;
                all += sh.peer_a[c];
            }
            run = a;
        };
        // The bin at which the running sum (from off) reaches goal, the sums before and with it: to every CTA.
        auto cross = [&](u64 goal, u64 own, u64 run, u64 off) {
            const u64 upto = off + run;
            if (tid < PER && upto - own < goal && goal <= upto)   // one thread of the cluster
                for (int c = 0; c < SMP_CL; c++) {
                    SmpShared* o = cl.map_shared_rank(&sh, c);
                    o->cut_bin = (uint32_t)(rank * PER + tid);
                    o->cut_a = upto - own;
                    o->cut_n = upto < 0xffffffffull ? (uint32_t)upto : 0xffffffffu;
                }
            cl.sync();
        };
        // This CTA's tokens of the given bins (level 0: `first`, else of the ranks lo .. hi) into its list; their
        // number in the cluster, and their first and last rank here.
        auto gather = [&](auto in_bin, u64& mn, u64& mxr) {
            mn = ~0ull;
            mxr = 0;
            for (int i = tid; i < n4; i += 4 * SMP_THREADS) {   // four reads in flight
                float4 v[4];
#pragma unroll
                for (int z = 0; z < 4; z++) {
                    const int at = i + z * SMP_THREADS;
                    v[z] = at < n4 ? *reinterpret_cast<const float4*>(x + 4 * at) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
                uint32_t hit = 0;
#pragma unroll
                for (int z = 0; z < 4; z++) {
                    const float l[4] = {v[z].x, v[z].y, v[z].z, v[z].w};
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (i + z * SMP_THREADS < n4 && in_bin(l[j], 4 * (i + z * SMP_THREADS) + j)) hit |= 1u << (4 * z + j);
                }
                while (hit) {
                    const int z = __ffs(hit) - 1;
                    hit &= hit - 1;
                    const u64 rk = rank_of(4 * (i + (z >> 2) * SMP_THREADS) + (z & 3));
                    mn = rk < mn ? rk : mn;
                    mxr = rk > mxr ? rk : mxr;
                    const uint32_t at = atomicAdd(&sh.n_cand, 1u);
                    if (at < SMP_CAND) sh.cand[at] = rk;
                }
            }
            __syncthreads();
            if (tid < SMP_CL) cl.map_shared_rank(&sh, tid)->peer_n[rank] = sh.n_cand;
            cl.sync();
            uint32_t m = 0;
#pragma unroll
            for (int c = 0; c < SMP_CL; c++) m += sh.peer_n[c];
            return m;
        };
        // In CTA 0: this thread's of the gathered tokens (0: none).
        auto candidate = [&] {
            int m = 0, from = -1, at = 0;   // number `at` of CTA `from`
#pragma unroll
            for (int c = 0; c < SMP_CL; c++) {
                const int nc = (int)sh.peer_n[c];
                if (tid >= m && tid < m + nc) {
                    from = c;
                    at = tid - m;
                }
                m += nc;
            }
            return from >= 0 ? cl.map_shared_rank(&sh, from)->cand[at] : 0ull;
        };
        // In CTA 0: the candidate at which the sum, from g, reaches goal; to every CTA.
        auto resolve = [&](u64 goal, bool counts, u64 g, int m) {
            const u64 me = candidate();
            bool in = me != 0;
            const u64 w = !in ? 0 : counts ? 1 : weight_of(smp_logit((uint32_t)(me >> 32)));
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
                const u64 own_n = sh.count[tid], own = (u64)sh.whi[tid] << 32 | sh.wlo[tid];
                const u64 a = smp_scan(own, sh.warp64);
                if (g + a - own < goal && goal <= g + a) {
                    sh.n_list = (uint32_t)own_n;
                    sh.cut_bin = (uint32_t)tid;
                    sh.tot_a = g + a - own;
                }
                __syncthreads();
                g = sh.tot_a;
                left = (int)sh.n_list;
                in = in && bin == (int)sh.cut_bin;
            }
            __syncthreads();
            if (tid == 0) sh.n_list = 0;
            __syncthreads();
            if (in) {
                const uint32_t to = atomicAdd(&sh.n_list, 1u);
                sh.last[to] = me;
                sh.cand_w[to] = w;
            }
            __syncthreads();
            if (warp == 0 && lane < left) {
                const u64 mine = sh.last[lane], mine_w = sh.cand_w[lane];
                u64 before = g;
                for (int j = 0; j < left; j++)
                    if (sh.last[j] > mine) before += sh.cand_w[j];
                if (before < goal && goal <= before + mine_w)
                    for (int c = 0; c < SMP_CL; c++) cl.map_shared_rank(&sh, c)->cut_rank = mine;
            }
        };

        // Rank at which the running sum reaches goal, from the crossed bin on.
        auto search = [&](u64 goal, bool counts, auto weigh) {
            const uint32_t bin = sh.cut_bin;
            u64 g = sh.cut_a, lo = 0, hi = ~0ull, mn, mxr;
            uint32_t m = gather([&](float l, int) { return bin_of(l) == (int)bin; }, mn, mxr);
            if (!counts && m <= SMP_CAND) {   // this CTA's kept weights: the bins before, and of this one the ranks from the cut on
                known = !(mp > 0.f);
                for (int i = tid; i < (int)bin; i += SMP_THREADS) own_kept += (u64)sh.whi[i] << 32 | sh.wlo[i];
            }
            while (m > SMP_CAND) {   // too many: bins over the ranks between the first and the last of them
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
                if (tid == 0) sh.n_cand = 0;
                lo = ~0ull;
                hi = 0;
#pragma unroll
                for (int i = 0; i < SMP_CL; i++) {
                    lo = sh.peer_a[i] < lo ? sh.peer_a[i] : lo;
                    hi = sh.peer_b[i] > hi ? sh.peer_b[i] : hi;
                }
                const int shift = max(0, 64 - __clzll(hi - lo) - 11);   // (hi - lo) >> shift < 2048
                clear();
                for (int i = tid; i < n; i += SMP_THREADS) {
                    const u64 rk = rank_of(i);
                    if (rk < lo || rk > hi) continue;
                    const int at = (int)((hi - rk) >> shift);
                    if (counts) atomicAdd(&sh.count[at], 1u);
                    else put(at, weigh(x[i], i));
                }
                u64 own, run, all;
                merge(counts, own, run, all);
                cross(goal, own, run, g);
                const uint32_t fine = sh.cut_bin;
                g = sh.cut_a;
                m = gather([&](float, int i) {
                    const u64 rk = rank_of(i);
                    return rk >= lo && rk <= hi && (uint32_t)((hi - rk) >> shift) == fine;
                }, mn, mxr);
            }
            if (rank == 0) resolve(goal, counts, g, (int)m);
            cl.sync();
            const u64 at = sh.cut_rank;
            if (known && tid < (int)sh.peer_n[rank] && sh.cand[tid] >= at)
                own_kept += weight_of(smp_logit((uint32_t)(sh.cand[tid] >> 32)));
            if (tid == 0) sh.n_cand = 0;
            return at;
        };
        u64 own, run, all;
        if (by_k) {
            for (int i = tid; i < n4; i += SMP_THREADS) {
                const float4 v = *reinterpret_cast<const float4*>(x + 4 * i);
                atomicAdd(&sh.count[bin_of(v.x)], 1u);
                atomicAdd(&sh.count[bin_of(v.y)], 1u);
                atomicAdd(&sh.count[bin_of(v.z)], 1u);
                atomicAdd(&sh.count[bin_of(v.w)], 1u);
            }
            merge(true, own, run, all);
            cross((u64)k, own, run, 0);
            const int bin = (int)sh.cut_bin;
            if (bin < SMP_BINS - 1 && sh.cut_n <= SMP_CAND) {   // few: CTA 0 ends it
                u64 mn, mxr;
                const int m = (int)gather([&](float l, int) { return bin_of(l) <= bin; }, mn, mxr);
                const u64 me = rank == 0 ? candidate() : 0;
                cl.sync();   // after this no CTA touches another's memory
                if (rank) return;
                const float e = me ? exp_of(smp_logit((uint32_t)(me >> 32))) : 0.f;
                const u64 w = me ? smp_weight(e) : 0;
                if (me) {
                    sh.cand[tid] = me;
                    sh.cand_w[tid] = w;
                }
                __syncthreads();
                int pos = 0;
                u64 before = 0;
                for (int j = 0; j < m; j++)
                    if (sh.cand[j] > me) {
                        pos++;
                        before += sh.cand_w[j];
                    }
                bool in = me && pos < k;
                if (by_p) {
                    const u64 goal = smp_share(block_sum(in ? w : 0), (uint32_t)rintf(fmaxf(p, 0.f) * 16777216.f));
                    in = in && (before < goal || pos == 0);
                }
                const u64 mine = in && e >= mp ? w : 0;
                __syncthreads();
                if (me) sh.cand_w[tid] = mine;
                const u64 target = smp_share(block_sum(mine), min((uint32_t)uf, 0xFFFFFFu));
                u64 upto = 0;   // kept weights of lower indices (larger complements)
                for (int j = 0; j < m; j++)
                    if ((uint32_t)sh.cand[j] > (uint32_t)me) upto += sh.cand_w[j];
                if (target >= upto && target < upto + mine) out[row] = (int)~(uint32_t)me;
                return;
            }
            // (the last bin's tokens have no weight: nothing is cut that could be drawn)
            if (bin < SMP_BINS - 1) cut = search((u64)k, true, [](float, int) { return 0ull; });
        }
        if (by_p) {
            // tokens that top-k left; all of them: the sum that the share is taken of
            auto weigh = [&](float l, int i) { return rank_of(i) >= cut ? weight_of(l) : 0ull; };
            if (by_k) clear();
            float4 v, next = make_float4(0.f, 0.f, 0.f, 0.f);   // read ahead of the atomics
            if (tid < n4) next = *reinterpret_cast<const float4*>(x + 4 * tid);
            for (int i = tid; i < n4; i += SMP_THREADS) {
                v = next;
                if (i + SMP_THREADS < n4) next = *reinterpret_cast<const float4*>(x + 4 * (i + SMP_THREADS));
                const float l[4] = {v.x, v.y, v.z, v.w};
                int bin[4];
                u64 w[4];
                uint32_t old[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    bin[j] = bin_of(l[j]);
                    w[j] = cut ? weigh(l[j], 4 * i + j) : weight_of(l[j]);
                }
                // four at once, so that the atomics' round trips overlap
#pragma unroll
                for (int j = 0; j < 4; j++) old[j] = bin[j] < SMP_BINS - 1 ? atomicAdd(&sh.wlo[bin[j]], (uint32_t)w[j]) : 0u;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t hi = (uint32_t)(w[j] >> 32) + (old[j] + (uint32_t)w[j] < old[j]);
                    if (hi) atomicAdd(&sh.whi[bin[j]], hi);
                }
            }
            merge(false, own, run, all);
            const u64 goal = smp_share(all, (uint32_t)rintf(fmaxf(p, 0.f) * 16777216.f));
            u64 c2;
            if (goal) {
                cross(goal, own, run, 0);
                c2 = search(goal, false, weigh);
            } else {
                c2 = (u64)smp_key(mx) << 32 | ~first_max();   // the first token alone
            }
            cut = c2 > cut ? c2 : cut;
        }
    }

    // ---- the draw, in index order: threads take consecutive runs of float4s,
    // each lane from another place of its run on (a warp's reads then fall on
    // different banks; whole numbers add up the same in any order)
    const int run = (n4 + SMP_THREADS - 1) / SMP_THREADS;
    const int r0 = min(tid * run, n4), r1 = min(r0 + run, n4);
    const float cut_l = cut ? smp_logit((uint32_t)(cut >> 32)) : -INFINITY;
    const uint32_t cut_i = cut ? ~(uint32_t)cut : 0xffffffffu;   // the last kept index of logit cut_l
    auto kept = [&](float l, int i, float& e) {   // token i after the filters
        e = exp_of(l);
        return (l > cut_l || (l == cut_l && (uint32_t)(i0 + i) <= cut_i)) && e >= mp;
    };
    u64 upto = 0, total = 0, sum = 0;   // kept weights before this CTA (then this thread), all, this thread's
    auto exchange = [&](u64 own) {
        if (tid < SMP_CL) cl.map_shared_rank(&sh, tid)->peer_sum[rank] = own;
        cl.sync();   // after this no CTA touches another's memory
#pragma unroll
        for (int c = 0; c < SMP_CL; c++) {
            if (c < rank) upto += sh.peer_sum[c];
            total += sh.peer_sum[c];
        }
        return smp_share(total, min((uint32_t)uf, 0xFFFFFFu));
    };
    u64 target = 0;
    if (known) {   // only the CTA that the target falls into looks for it
        const u64 own = block_sum(own_kept);
        target = exchange(own);
        if (target < upto || target >= upto + own) return;
    }
    {
        uint32_t h = 0;   // at most 2^17 x 2^15 / 512 x 2
        int lo = 0;
        int i = r0 + lane % max(run, 1);
#pragma unroll 2
        for (int step = 0; step < run; step++) {
            const float4 v = i < r1 ? *reinterpret_cast<const float4*>(x + 4 * i)
                                    : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= cut_l) {
                const float l[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float e;
                    uint32_t eh;
                    int el;
                    const bool in = kept(l[j], 4 * i + j, e);
                    smp_parts(e, eh, el);
                    h += in ? eh : 0u;
                    lo += in ? el : 0;
                }
            }
            i = i + 1 == r0 + run ? r0 : i + 1;
        }
        sum = smp_join(h, lo);
    }
    const u64 incl = smp_scan(sum, sh.warp64);   // running sums over the block
    if (!known) {
        if (tid == SMP_THREADS - 1) sh.tot_a = incl;
        __syncthreads();
        target = exchange(sh.tot_a);
    }
    upto += incl - sum;
    // the thread whose run holds the target; its warp looks through the run
    const uint32_t who = __ballot_sync(0xffffffffu, target >= upto && target < upto + sum);
    if (!who) return;
    const int src_lane = __ffs(who) - 1;
    u64 at = __shfl_sync(0xffffffffu, upto, src_lane);
    const int f0 = 4 * __shfl_sync(0xffffffffu, r0, src_lane), f1 = 4 * __shfl_sync(0xffffffffu, r1, src_lane);
    for (int i = f0; i < f1; i += 32) {
        float e;
        u64 c = 0;
        if (i + lane < f1 && kept(x[i + lane], i + lane, e)) c = smp_weight(e);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, c, o);
            if (lane >= o) c += y;
        }
        const uint32_t m = __ballot_sync(0xffffffffu, at + c > target);
        if (m) {
            if (lane == 0) out[row] = i0 + i + __ffs(m) - 1;
            return;
        }
        at += __shfl_sync(0xffffffffu, c, 31);
    }
}

}  // namespace gb

extern "C" int gb_sample(const float* logits, int ldl, int rows, int vocab, const float* temperature, const int* top_k,
                         const float* top_p, const float* min_p, const float* u, int* out, void* stream) {
    if (rows < 0 || vocab <= 0 || ldl < vocab) return GB_EINVAL;
    if (vocab > GB_SAMPLE_MAX_VOCAB) return GB_ELIMIT;
    if (rows == 0) return GB_OK;
    if (!logits || !u || !out) return GB_EINVAL;
    if (rows > 0x7fffffff / gb::SMP_CL) return GB_ELIMIT;
    const int slice = ((vocab + gb::SMP_CL - 1) / gb::SMP_CL + 3) / 4 * 4;
    const size_t smem = (sizeof(gb::SmpShared) + 15) / 16 * 16 + (size_t)slice * sizeof(float);
    constexpr size_t most = (sizeof(gb::SmpShared) + 15) / 16 * 16 + (size_t)GB_SAMPLE_MAX_VOCAB / gb::SMP_CL * sizeof(float);
    static_assert(most <= 227 * 1024, "shared memory");
    if (gb::set_smem_once(reinterpret_cast<const void*>(gb::k_sample), (int)most) != cudaSuccess) return GB_ECUDA;
    // More rows than two CTAs an SM take at once: those that need a search first.
    // Five kinds of settings by turns, without / with; all rows top-p (us):
    //   vocabulary 32,000    38 rows 17 / 15, 26 / 28     100 rows 32 / 32, 48 / 52
    //              64,000    61      28 / 24, 40 / 42     100      41 / 37, 65 / 69
    //              96,000   100      58 / 51, 85 / 89     148      77 / 72, 117 / 123
    //             128,256   100      68 / 59, 99 / 103    148      90 / 83, 136 / 142
    // It gains where rows are long and few: a row per 800 tokens, at most four
    // times as many as run at once.
    const int at_once = 2 * gb::sm_count() / gb::SMP_CL;
    const bool longest_first = (temperature || top_k || top_p) && rows > at_once && rows <= 4 * at_once &&
                               rows <= vocab / 800 && rows <= gb::SMP_THREADS;
    return gb::launch_pdl(gb::k_sample, dim3(rows * gb::SMP_CL), gb::SMP_THREADS, (int)smem,
                          static_cast<cudaStream_t>(stream), logits, ldl, vocab, slice, temperature, top_k, top_p, min_p,
                          u, out, longest_first) == cudaSuccess
               ? GB_OK
               : GB_ECUDA;
}
