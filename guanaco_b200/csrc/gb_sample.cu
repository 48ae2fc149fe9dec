// gb_sample.cu -- one token per row of logits: temperature, top-k, top-p,
// min-p, drawn with a given random number.
//
// The weights are integers, w = rint(2^40 e), e = exp((l - max) / T) in fp32,
// so every sum is exact and the token does not depend on how the row is split.
// Every filter keeps a prefix of the order (logit descending, index
// ascending), so a cut is a logit key and a number of equal logits that are
// kept, lowest index first: found by radix selection over the keys, with the
// digits' counts (top-k) or weights (top-p).
//
// One CTA per row; the row is read again for each pass.
#include "gb_common.cuh"
#include "gb_internal.h"

namespace gb {

constexpr int SMP_THREADS = 1024;
typedef unsigned long long u64;

// Order-preserving key of a logit: larger logits have larger keys, NaN is
// -inf and -0 is +0.
__device__ __forceinline__ uint32_t smp_key(float l) {
    if (l != l) l = -INFINITY;
    const uint32_t b = __float_as_uint(l + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float smp_logit(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ float smp_exp(float l, float mx, float t) {
    return l == mx ? 1.f : expf(__fdiv_rn(l - mx, t));   // mx may be +inf: the others weigh nothing
}
__device__ __forceinline__ u64 smp_weight(float e) { return __float2ull_rn(e * 1099511627776.f); }
// floor(total * part / 2^24), part <= 2^24
__device__ __forceinline__ u64 smp_share(u64 total, uint32_t part) {
    return (total >> 24) * part + (((total & 0xFFFFFFull) * part) >> 24);
}

template <typename T, typename F>
__device__ T block_reduce(T v, F f, T* sh) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[threadIdx.x & 31];
#pragma unroll
    for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

__global__ void __launch_bounds__(SMP_THREADS)
k_sample(const float* __restrict__ logits, int ldl, int vocab, const float* __restrict__ temperature,
         const int* __restrict__ top_k, const float* __restrict__ top_p, const float* __restrict__ min_p,
         const float* __restrict__ uu, int* __restrict__ out) {
    __shared__ u64 hist[256], sh64[32];
    __shared__ uint32_t sh32[32];
    __shared__ u64 s_gt, s_bin;
    __shared__ uint32_t s_digit;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float* x = logits + (size_t)r * ldl;
    auto vmax = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    auto vmin = [](uint32_t a, uint32_t b) { return a < b ? a : b; };
    auto add = [](u64 a, u64 b) { return a + b; };

    uint32_t kmax = 0;
    for (int i = tid; i < vocab; i += SMP_THREADS) kmax = vmax(kmax, smp_key(x[i]));
    kmax = block_reduce(kmax, vmax, sh32);
    const float mx = smp_logit(kmax);
    if (mx == -INFINITY) {
        if (tid == 0) out[r] = -1;
        return;
    }
    const float t = temperature ? temperature[r] : 1.f;
    if (!(t > 0.f)) {
        uint32_t first = 0xffffffffu;
        for (int i = tid; i < vocab; i += SMP_THREADS)
            if (smp_key(x[i]) == kmax) first = vmin(first, (uint32_t)i);
        first = block_reduce(first, vmin, sh32);
        if (tid == 0) out[r] = (int)first;
        return;
    }
    const int k = top_k ? top_k[r] : 0;
    const float p = top_p ? top_p[r] : 1.f;
    const float mp = min_p && min_p[r] > 0.f ? fminf(min_p[r], 1.f) : 0.f;

    // kept so far: key > cut, and the first `ties` indices of key == cut
    uint32_t cut = 0, ties = 0xffffffffu;
    // Finds the digit string of the first key, from the top, at which the
    // running sum of `what` (1 or the weight) reaches `goal` >= 1; `gt` = the
    // sum above it.
    auto select = [&](u64 goal, bool count, u64& gt, u64& at) {
        uint32_t prefix = 0;
        gt = 0;
        for (int sft = 24; sft >= 0; sft -= 8) {
            __syncthreads();
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < vocab; i += SMP_THREADS) {
                const uint32_t key = smp_key(x[i]);
                if (sft < 24 && (key >> (sft + 8)) != prefix) continue;
                if (!count && key < cut) continue;
                const u64 w = count ? 1ull : smp_weight(smp_exp(smp_logit(key), mx, t));
                if (w) atomicAdd(&hist[(key >> sft) & 255], w);
            }
            __syncthreads();
            if (tid == 0) {
                u64 g = gt;
                int dgt = 255;
                for (; dgt > 0; dgt--) {
                    if (g + hist[dgt] >= goal) break;
                    g += hist[dgt];
                }
                s_gt = g;
                s_digit = dgt;
                s_bin = hist[dgt];
            }
            __syncthreads();
            gt = s_gt;
            prefix = (prefix << 8) | s_digit;
        }
        at = s_bin;   // sum at the key itself
        return prefix;
    };
    if (k > 0 && k < vocab) {
        u64 gt, at;
        cut = select((u64)k, true, gt, at);
        ties = (uint32_t)((u64)k - gt);
    }
    if (p < 1.f) {
        u64 gt, at, total = 0;
        for (int i = tid; i < vocab; i += SMP_THREADS) {
            const uint32_t key = smp_key(x[i]);
            if (key > cut || (key == cut && ties == 0xffffffffu)) total += smp_weight(smp_exp(smp_logit(key), mx, t));
        }
        total = block_reduce(total, add, sh64);
        const u64 wcut = smp_weight(smp_exp(smp_logit(cut), mx, t));
        if (ties != 0xffffffffu) total += ties * wcut;
        const u64 goal = smp_share(total, (uint32_t)rintf(fmaxf(p, 0.f) * 16777216.f));
        if (goal == 0) {
            cut = kmax;
            ties = 1;
        } else {
            cut = select(goal, false, gt, at);
            const u64 w = smp_weight(smp_exp(smp_logit(cut), mx, t));
            const u64 need = goal - gt;   // the j-th tie is kept while j w < need
            ties = (uint32_t)((need + w - 1) / w);
        }
    }
    // ---- the draw, in index order: warps take consecutive runs of indices
    const int run = (vocab + SMP_THREADS / 32 - 1) / (SMP_THREADS / 32);
    const int i0 = min(warp * run, vocab), i1 = min(i0 + run, vocab);
    // ties before this warp's run
    uint32_t eq = 0;
    for (int i = i0 + lane; i < i1; i += 32) eq += smp_key(x[i]) == cut;
    eq = __reduce_add_sync(0xffffffffu, eq);
    __syncthreads();
    if (lane == 0) sh32[warp] = eq;
    __syncthreads();
    uint32_t before = 0;
    for (int w = 0; w < warp; w++) before += sh32[w];
    auto weight_at = [&](int i, uint32_t& seen) {   // weight of index i after the filters; seen: ties before the warp's step
        const uint32_t key = i < i1 ? smp_key(x[i]) : 0u;
        const bool tie = i < i1 && key == cut;
        const uint32_t m = __ballot_sync(0xffffffffu, tie);
        const uint32_t at = seen + __popc(m & ((1u << lane) - 1));
        seen += __popc(m);
        if (i >= i1 || key < cut || (tie && at >= ties)) return 0ull;
        const float e = smp_exp(smp_logit(key), mx, t);
        return e >= mp ? smp_weight(e) : 0ull;
    };
    u64 sum = 0;
    uint32_t seen = before;
    for (int i = i0; i < i1; i += 32) sum += weight_at(i + lane, seen);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sh64[warp] = sum;
    __syncthreads();
    u64 upto = 0, total = 0;
    for (int w = 0; w < SMP_THREADS / 32; w++) {
        if (w < warp) upto += sh64[w];
        total += sh64[w];
    }
    const float uf = fminf(fmaxf(uu[r], 0.f), 1.f) * 16777216.f;
    const u64 target = smp_share(total, min((uint32_t)uf, 0xFFFFFFu));
    if (target < upto || target >= upto + sh64[warp]) return;
    seen = before;
    for (int i = i0; i < i1; i += 32) {   // the run that holds the target: find the index
        const u64 w = weight_at(i + lane, seen);
        u64 c = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, c, o);
            if (lane >= o) c += y;
        }
        const uint32_t m = __ballot_sync(0xffffffffu, upto + c > target);
        if (m) {
            if (lane == 0) out[r] = i + __ffs(m) - 1;
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
    gb::k_sample<<<rows, gb::SMP_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(logits, ldl, vocab, temperature, top_k,
                                                                               top_p, min_p, u, out);
    return cudaGetLastError() == cudaSuccess ? GB_OK : GB_ECUDA;
}
