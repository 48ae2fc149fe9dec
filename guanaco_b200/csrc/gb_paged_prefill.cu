// gb_paged_prefill.cu -- causal attention of packed prompts over the paged
// KV cache, on the tcgen05 tensor cores.
//
// A CTA takes one KV head and 2 x 128 rows of one sequence: row = (query,
// query head of the group), 128 / group queries a tile, so that a K / V tile
// read from the cache serves every head that shares it.  Keys come in tiles of
// NK.  For each of the two row tiles, alternately:
//   S = Q K^T    A = Q, B = K, both K-major in shared memory (128-byte swizzle)
//   softmax      a thread takes one row (= tensor-memory lane) or half of its
//                keys: scale, causal mask, running maximum and sum; P = 2^(x - m)
//                back into tensor memory over S
//   O += P V     A = P from tensor memory, B = V as it lies in the cache (rows
//                = keys, MN-major): V is never transposed
// While one row tile's softmax runs the tensor cores work for the other.  With
// one product per operand and tiles of 64 keys there is room for two buffers of
// S, so the next scores are there when a softmax ends.  With several products
// (fp32 activations, a Q8_0 cache) the tensor cores are the bound, and Q (its
// high parts) is kept in tensor memory, which takes its reads off shared
// memory.  Two threads per row only exchange a vote per key tile.
// The maximum moves only when a score exceeds it by more than PP_TAU (log2
// units), so O in tensor memory is rarely rescaled.
//
// Precision.  P is rounded to fp16 for fp16 activations (an error of the size of
// the fp16 output's own rounding); for fp32 ones Q (scaled by a power of two per
// row) and P are split into an fp16 value and an fp16 remainder.  Q8_0 values
// (code x scale has 18 bits) are always split so, a product for each part:
// hi.hi + lo.hi + hi.lo for fp32, hi.hi + hi.lo for fp16.  (K and V rounded to
// fp16 instead: error against 64 bits 4.0e-4, that of the output's rounding alone 2.1e-4,
// and 91 us; split 2.8e-4 and 106 us; five prompts of up to 968 tokens.)
//
// The tensor cores' additions truncate, always towards zero: their sums come
// out low.  fp32 adds the products with remainders into S first, so that the
// truncations are of their size, keeps those of P V apart where there is room
// (hd 64), and starts O anew every FLUSH tiles, adding what was there, rounded
// to nearest, to a running sum in the workspace (L2-resident, 128 KB per SM).
// Error against 64 bits of five prompts of up to 968 tokens in Q8_0 (plain fp32
// in another order 8.6e-7) and time, hd 128: every 16 tiles 2.3e-6, 175 us; 8
// 1.7e-6; 4 1.2e-6, 194 us; 2 8.9e-7, 211 us; hd 64 (6.7e-7): 16 8.9e-7; 8 7.2e-7;
// 4 5.6e-7.  Never, with the remainders last: 1.1e-5 on 8192 tokens.
//
// An F16 cache's tiles are TMA copies, one box per page and 64 columns; Q8_0
// tiles are dequantised by four warps, a row per thread.  Rows past the last
// key are zeroed in V (stale cache rows may hold anything).
//
// Rows whose result is not finite are computed once more by a warp each, from
// the definition in fp32 (pp_row): P V also runs over the keys that a row does
// not see, where an infinity or no number times the weight 0 is no number, and
// an infinite K times q's two parts, or a Q8_0 value beyond 65504 as two halves,
// may be none although the score or the value is a number.  Finite inputs of
// ordinary size never come here.  One prompt of 8192, fp16, F16 cache, with an
// infinity in V at the first position (each row rightly shows it: found at
// once) 1.05 ms instead of 0.48, at the last (the 256 rows of 8 CTAs that it
// spoils: 8192 keys each) 20.8 ms.
//
// Few rows over a long axis: the host cuts the keys over gridDim.y CTAs, which
// leave (m, l, O) partials; the last to arrive joins them in order.
//
// 32 / 8 heads of 128, in a CUDA graph: one prompt of 8192, fp16, F16 cache 474-487
// us, 1130-1160 TFLOP/s (a call among others 552-562 us, under the power cap), where
// the exponentials and the tensor cores take turns; five prompts of up to 968, fp32,
// Q8_0 147-151 us, 231 TFLOP/s of three products: the tensor cores, 2300 cycles for
// 128 rows and 64 keys, and 30,000 cycles a CTA before and after them.
#include "gb_mt.cuh"
#include "gb_paged.cuh"
#include "gb_tc.cuh"

#include <cuda.h>

namespace gb {

constexpr int PP_POLY = 8;                      // of this many pairs of exponentials one is a polynomial
constexpr float PP_TAU = 8.f, PP_LIFT = 6.f;   // p <= 2^14; small p stay normal fp16 numbers
constexpr int PP_SPLIT = 4;                     // key tiles at least of a CTA where keys are split
constexpr int PP_SMEM_MAX = 227 * 1024 - 4096;  // less alignment slack and static shared memory

template <typename A, int HD, int DT>
struct PpCfg {
    static constexpr bool F32 = sizeof(A) == 4, Q8 = DT == GB_DT_Q8_0;
    // fp16, F16 cache, hd 128: tiles of 128 keys (an MMA of N 128 takes 80 cycles,
    // one of N 64 takes 64), one buffer of S, two threads per row; hd 64: 64 keys,
    // two buffers and one thread per row.  One prompt of 8192 tokens that way /
    // the other, when this was chosen: hd 128 489 / 597 us, hd 64 580 / 449 us.  Several products per
    // operand: one buffer, two threads per row (Q8_0 hd 128 896 us, with two
    // buffers and Q in shared memory 1543 us).
    static constexpr bool WIDE = !F32 && !Q8 && HD == 128;
    static constexpr int NK = WIDE ? 128 : 64;         // keys per tile
    static constexpr int KS = Q8 ? 2 : 1;              // fp16 parts of K and V (of Q and P: 2 for fp32)
    static constexpr int G = HD / 64;                  // 64-column groups (128 bytes)
    static constexpr int QB = 128 * HD * 2;            // bytes of a row tile's part
    static constexpr int KB = NK * HD * 2;             // bytes of a K (or V) tile's part
    static constexpr int ST0 = (PP_SMEM_MAX - 2 * QB) / (2 * KS * KB);
    static constexpr int ST = ST0 > 4 ? 4 : ST0;       // K / V stages
    static constexpr int SMEM = 2 * QB + ST * 2 * KS * KB + 1024;
    // producer warps; fp32 at hd 64: two leave every thread 96 registers instead of
    // 80 (five prompts of up to 968 tokens 107 / 113 us; hd 128, twice the rows' bytes, 224 / 193 us)
    static constexpr int PROD = !Q8 ? 1 : F32 && HD == 64 ? 2 : 4;
    static constexpr bool QT = F32 || Q8;              // Q, or its high parts, in tensor memory
    static constexpr int TR = QT || WIDE ? 2 : 1;      // softmax threads per row
    static constexpr int SOFT = 256 * TR, MMA = SOFT / 32;   // their number; the MMA warp
    static constexpr int THREADS = SOFT + 32 + PROD * 32;
    // tensor memory columns: S (and P over it) of row tile i at SW i, in NS
    // buffers; fp32: Q's high parts at 128 + 64 i; O at 256 + 128 i
    static constexpr int NS = QT || WIDE ? 1 : 2;      // buffers of S
    static constexpr uint32_t SW = NK * NS;
    static constexpr uint32_t PLO = NK / 4;            // fp32: P's remainders, from a part's first column
    static constexpr int NH = NK / TR;                 // keys of a softmax thread
    static constexpr uint32_t OS = F32 && HD == 64 ? 64 : 0;   // there is room for O's small products, from O's first column
    static constexpr int FLUSH = OS ? 8 : 4;           // fp32: key tiles whose P V stay in tensor memory
    static_assert(ST >= 2, "shared memory");
};

struct PpArgs {
    PagedView c;
    BatchView b;
    const void* q;
    void* out;
    int ldq, ldo, group, bq;      // bq: queries per row tile
    float* part;
    unsigned* tickets;
    unsigned* err;
};

__device__ __forceinline__ float pp_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^x of a pair without the special function unit, whose 16 results a cycle
// bound the kernel: x = j + r, j the nearest integer, 2^r by the degree-4
// polynomial of least relative error on [-1/2, 1/2] (2.6e-6, a hundredth of
// P's rounding), j added to the exponent.  x is kept above -126; one that is no
// number (0x7fffffff through all of it) comes out as the largest float, an
// infinity as a half, so its row's output is not finite.
__device__ __forceinline__ float pp_max_nan(float a, float b) {   // no number if either is none
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float2 pp_ex2_poly(float2 x) {
    x.x = pp_max_nan(x.x, -126.f);
    x.y = pp_max_nan(x.y, -126.f);
    const float2 big = make_float2(12582912.f, 12582912.f);   // 1.5 2^23: adding it rounds to an integer
    const float2 t = __fadd2_rn(x, big);
    const float2 j = __fadd2_rn(t, make_float2(-12582912.f, -12582912.f));
    const float2 r = __fadd2_rn(x, make_float2(-j.x, -j.y));
    float2 y = __ffma2_rn(make_float2(0.009570086f, 0.009570086f), r, make_float2(0.05591785f, 0.05591785f));
    y = __ffma2_rn(y, r, make_float2(0.24024744f, 0.24024744f));
    y = __ffma2_rn(y, r, make_float2(0.6931218f, 0.6931218f));
    y = __ffma2_rn(y, r, make_float2(0.9999993f, 0.9999993f));
    return make_float2(__uint_as_float(__float_as_uint(y.x) + (__float_as_uint(t.x) << 23)),
                       __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(t.y) << 23)));
}
__device__ __forceinline__ uint32_t pp_pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Among the 256 threads of a row tile with two threads per row (barrier id): a vote, a barrier.
__device__ __forceinline__ bool pp_vote(int id, bool v) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.aligned.pred q, %2, 256, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"((uint32_t)v), "r"(id)
        : "memory");
    return any != 0;
}
__device__ __forceinline__ void pp_sync(int id) { asm volatile("barrier.cta.sync.aligned %0, 256;" ::"r"(id) : "memory"); }
// Byte offset of the 16-byte unit u (8 halves) of row r in a swizzled tile of R rows.
__device__ __forceinline__ uint32_t pp_off(int r, int u, int R) {
    return (uint32_t)((u >> 3) * R * 128 + r * 128 + (((u ^ r) & 7) << 4));
}

// N (2, 4, 8) columns from col on, a multiple of N, of row r of a slab.
template <int HD, int DT, int N>
__device__ __forceinline__ void pp_cached(const uint8_t* slab, int shift, int r, int col, float (&x)[N]) {
    constexpr int B = DT == GB_DT_F16 ? 2 * N : N;   // bytes
    const uint8_t* p = slab + ((size_t)r * HD + col) * (B / N);
    uint32_t w[B < 4 ? 1 : B / 4];
    if constexpr (B == 16) {
        const uint4 y = ldg4(p);
        w[0] = y.x; w[1] = y.y; w[2] = y.z; w[3] = y.w;
    } else if constexpr (B == 8) {
        const uint2 y = __ldg(reinterpret_cast<const uint2*>(p));
        w[0] = y.x; w[1] = y.y;
    } else if constexpr (B == 4) {
        w[0] = ldg1(p);
    } else {
        w[0] = ldg_u16(p);
    }
    if constexpr (DT == GB_DT_F16) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i / 2]));
            x[i] = f.x;
            x[i + 1] = f.y;
        }
    } else {
        const float d = __half2float(__ldg(reinterpret_cast<const __half*>(slab + ((size_t)HD << shift)) + r * (HD / 32) + col / 32));
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = d * (float)(int8_t)(w[i / 4] >> (8 * (i % 4)) & 0xffu);
    }
}
// Head h of token t, which sees the first n keys of sequence seq (none: zeros),
// whose output is not finite: one warp, 32 keys at a time, HD / 32 columns a lane.  Once the columns that are not finite are so
// here too, the output is left as it is: its other columns are right.
template <typename A, int HD, int DT>
__device__ __noinline__ void pp_row(const PpArgs& a, int seq, int kvh, int t, int h, int n) {
    constexpr int CO = HD / 32, V = 8;   // columns of a lane, rows in flight (of one page)
    const int lane = threadIdx.x & 31, col = lane * CO, rows = 1 << a.c.shift;
    const PagedView& c = a.c;
    const A* q = static_cast<const A*>(a.q) + (size_t)t * a.ldq + (size_t)h * HD + col;
    A* dst = static_cast<A*>(a.out) + (size_t)t * a.ldo + (size_t)h * HD + col;
    const float sc = 1.4426950408889634f / sqrtf((float)HD);
    float qx[CO], o[CO], m = -INFINITY, l = 0.f;   // l: of this lane's keys
    bool odd[CO];
#pragma unroll
    for (int i = 0; i < CO; i++) {
        qx[i] = (float)q[i];
        o[i] = 0.f;
        odd[i] = !isfinite((float)dst[i]);
    }
#pragma unroll 1
    for (int key0 = 0; key0 < n; key0 += 32) {
        const int key = min(key0 + lane, n - 1);
        const size_t slab = (size_t)max(page_of(c, a.b, seq, key, a.err), 0) * c.page_bytes + (size_t)kvh * c.slab;
        float x = 0.f;
        // a row's columns over the lanes, V rows in flight; lane j gets the sum of key j
#pragma unroll 1
        for (int j0 = 0; j0 < min(32, n - key0); j0 += V) {
            const uint8_t* at = c.k + __shfl_sync(0xffffffffu, slab, j0);
            float k[V][CO], s[V];
#pragma unroll
            for (int j = 0; j < V; j++)
                pp_cached<HD, DT, CO>(at, c.shift, min(key0 + j0 + j, n - 1) & (rows - 1), col, k[j]);
#pragma unroll
            for (int j = 0; j < V; j++) {
                s[j] = 0.f;
#pragma unroll
                for (int i = 0; i < CO; i++) s[j] = fmaf(qx[i], k[j][i], s[j]);
            }
            // halves of the lanes exchange halves of the keys, three times
#pragma unroll
            for (int w = V / 2; w; w >>= 1) {
                const bool up = lane & (w * (32 / V));
#pragma unroll
                for (int j = 0; j < w; j++) {
                    const float give = up ? s[j] : s[j + w], keep = up ? s[j + w] : s[j];
                    s[j] = keep + __shfl_xor_sync(0xffffffffu, give, w * (32 / V));
                }
            }
            s[0] += __shfl_xor_sync(0xffffffffu, s[0], 1);
            s[0] += __shfl_xor_sync(0xffffffffu, s[0], 2);
            const float y = __shfl_sync(0xffffffffu, s[0], (lane % V) * (32 / V));
            if (lane / V == j0 / V) x = y;
        }
        x = key0 + lane < n ? x * sc : -INFINITY;
        const float mn = fmaxf(m, warp_max(x)), ref = mn == -INFINITY ? 0.f : mn, al = pp_ex2(m - ref);   // 0 before the first finite score
        const float p = pp_ex2(x - ref);
        m = mn;
        l = fmaf(l, al, p);
#pragma unroll
        for (int i = 0; i < CO; i++) o[i] *= al;
#pragma unroll 1
        for (int j0 = 0; j0 < min(32, n - key0); j0 += V) {
            const uint8_t* at = c.v + __shfl_sync(0xffffffffu, slab, j0);
            float v[V][CO];
#pragma unroll
            for (int j = 0; j < V; j++)
                pp_cached<HD, DT, CO>(at, c.shift, min(key0 + j0 + j, n - 1) & (rows - 1), col, v[j]);
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float w = __shfl_sync(0xffffffffu, p, j0 + j);
#pragma unroll
                for (int i = 0; i < CO; i++)
                    if (key0 + j0 + j < n) o[i] = fmaf(w, v[j][i], o[i]);
            }
        }
        bool same = true;
#pragma unroll
        for (int i = 0; i < CO; i++) same = same && (!odd[i] || !isfinite(o[i]));
        if (__all_sync(0xffffffffu, same)) return;
    }
    l = warp_sum(l);
#pragma unroll
    for (int i = 0; i < CO; i++) dst[i] = (A)(n <= 0 ? 0.f : m == -INFINITY ? NAN : o[i] / l);
}

template <typename A, int HD, int DT>
__global__ void __launch_bounds__((PpCfg<A, HD, DT>::THREADS), 1)
k_paged_prefill(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                const __grid_constant__ PpArgs a) {
    using C = PpCfg<A, HD, DT>;
    constexpr int NK = C::NK, ST = C::ST;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* qs = sm;                                   // [2 tiles]: Q, for fp32 its remainders
    uint8_t* ks = sm + 2 * C::QB;                       // [ST][KS]
    uint8_t* vs = ks + ST * C::KS * C::KB;              // [ST][KS]
    __shared__ __align__(8) uint64_t bars[4 * ST + 14];
    __shared__ float s_row[2][2][128];                  // what the two threads of a row exchange
    __shared__ uint32_t tmem_slot;
    __shared__ int s_seq, s_blk, s_slot;
    __shared__ bool s_claimed;
    __shared__ unsigned s_last, s_again[8];             // s_again: rows whose result is not finite
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const PagedView& c = a.c;
    const BatchView& b = a.b;
    const int kvh = blockIdx.x % c.n_kv, y = blockIdx.x / c.n_kv;

    const uint32_t b0 = tc::smem_u32(&bars[0]);
    const uint32_t kfull = b0, kfree = b0 + 8 * ST, vfull = b0 + 16 * ST, vfree = b0 + 24 * ST;   // [ST] each
    const uint32_t sfull = b0 + 32 * ST, pfull = sfull + 32, odone = sfull + 64, ofull = sfull + 80, tail = sfull + 96, qread = sfull + 104;   // [2][2], [2][2], [2], [2], 1, 1
    if (tid == 32) {
        for (int i = 0; i < ST; i++) {
            mbs_init(kfull + 8 * i, C::PROD);
            mbs_init(kfree + 8 * i, 1);
            mbs_init(vfull + 8 * i, C::PROD);
            mbs_init(vfree + 8 * i, 1);
        }
        for (int i = 0; i < 4; i++) {   // [row tile][buffer]; P with two threads per row: [row tile][half]
            mbs_init(sfull + 8 * i, 1);
            mbs_init(pfull + 8 * i, 4);
        }
        for (int i = 0; i < 2; i++) {
            mbs_init(odone + 8 * i, 1);   // every P V of a row tile
            mbs_init(ofull + 8 * i, 1);   // its last
        }
        mbs_init(tail, 1);
        mbs_init(qread, C::MMA);          // Q's high parts have left the V stages
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid < 8) s_again[tid] = 0u;
    griddep_wait();   // launched ahead of the kernel before it
    // ---- which sequence and query block.  Up to 32 sequences: the y-th of all
    // blocks by their key tiles, the longest first; more: the sequences in order
    if (warp == 0) {
        if (lane == 0) s_seq = -1;
        __syncwarp();
        const int bb = 2 * a.bq;
        auto queries = [&](int s) { return s >= b.n_seq ? 0 : b.cu ? max(__ldg(b.cu + s + 1) - __ldg(b.cu + s), 0) : 1; };
        if (b.n_seq <= 32) {
            const int n = queries(lane), nb = (n + bb - 1) / bb, pos = n ? seq_len(b, lane, a.err) - n : 0;
            // blocks of this lane's sequence with at least t key tiles: their keys end past (t - 1) NK
            auto count = [&](int t) {
                if (t <= 0) return nb;
                const int past = (t - 1) * NK + 1 - pos;   // queries of the sequence before the first such block's end
                return past > n ? 0 : nb - max((past + bb - 1) / bb - 1, 0);
            };
            int lo = 0, hi = __reduce_max_sync(0xffffffffu, n ? max(pos + n + NK - 1, 0) / NK : 0) + 1;
            if (y < __reduce_add_sync(0xffffffffu, nb)) {
                while (hi - lo > 1) {   // more than y blocks have lo tiles, at most y have hi
                    const int mid = (lo + hi) >> 1;
                    if (__reduce_add_sync(0xffffffffu, count(mid)) > y) lo = mid;
                    else hi = mid;
                }
                const int longer = count(hi), same = count(lo) - longer;
                int incl = same;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += v;
                }
                const int at = y - __reduce_add_sync(0xffffffffu, longer) - (incl - same);
                if (at >= 0 && at < same) {
                    s_seq = lane;
                    s_blk = nb - 1 - longer - at;
                }
            }
        } else {
            int base = 0;
            for (int s0 = 0; s0 < b.n_seq; s0 += 32) {
                const int nb = (queries(s0 + lane) + bb - 1) / bb;
                int incl = nb;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += v;
                }
                const unsigned hit = __ballot_sync(0xffffffffu, y < base + incl);
                if (hit) {
                    if (lane == __ffs(hit) - 1) {
                        s_seq = s0 + lane;
                        s_blk = nb - 1 - (y - (base + incl - nb));
                    }
                    break;
                }
                base += __shfl_sync(0xffffffffu, incl, 31);
            }
        }
    }
    __syncthreads();
    const int seq = s_seq;
    if (seq < 0) return;
    const int t_begin = b.cu ? __ldg(b.cu + seq) : seq, t_end = min(b.cu ? __ldg(b.cu + seq + 1) : seq + 1, b.n_tokens);
    const int n_q = t_end - t_begin;
    const int q0 = s_blk * 2 * a.bq;
    if (q0 >= n_q || t_begin < 0) return;
    const int len = seq_len(b, seq, a.err);
    const int pos0 = len - n_q;                          // position of the first query (may be negative)
    const bool two = q0 + a.bq < n_q;                    // the second row tile has queries
    const int kend = len == 0 ? 0 : pos0 + min(q0 + 2 * a.bq, n_q);   // keys 0 .. kend - 1
    const int nt_all = kend > 0 ? (kend + NK - 1) / NK : 0;
    // keys split over gridDim.y CTAs, but at least PP_SPLIT tiles a CTA: the host knows the table's width alone
    const int per = gridDim.y == 1 ? nt_all : max(PP_SPLIT, (int)((nt_all + gridDim.y - 1) / gridDim.y));
    const int n_split = nt_all > 0 ? (nt_all + per - 1) / per : 1;
    if ((int)blockIdx.y >= n_split) return;
    const int j0 = blockIdx.y * per, nt = min(per, nt_all - j0);   // this CTA's key tiles j0 ..
    // the first row tile's queries may end before the last key tiles
    const int kend0 = max(pos0 + min(q0 + a.bq, n_q), 0);
    const int nt0 = min(nt, max((kend0 + NK - 1) / NK - j0, 0));

    // ---- rows
    constexpr int TR = C::TR, NH = C::NH, NS = C::NS;
    const int rt = warp / (4 * TR), hf = (warp >> 2) % TR, r = tid & 127;   // softmax threads: row tile, part, row
    const int qi = q0 + rt * a.bq + r / a.group, h = kvh * a.group + r % a.group;
    const bool live = warp < C::MMA && r < a.bq * a.group && qi < n_q;
    if (nt_all == 0) {   // nothing to see
        if (live) {
            A* dst = static_cast<A*>(a.out) + (size_t)(t_begin + qi) * a.ldo + (size_t)h * HD;
            const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            for (int d = hf * (HD / TR); d < (hf + 1) * (HD / TR); d += 8) act_store8(dst + d, z);
        }
        return;
    }

    // Where fp32 keeps a running sum: as many CTAs as places have one each; of
    // more, no more than SMs run at a time (a CTA takes all of an SM's tensor
    // memory), so that a free place is found from the SM's number on.
    const bool claim = C::F32 && (size_t)gridDim.x * gridDim.y > GB_MAX_SMS && nt > C::FLUSH;
    auto start_sync = [&] {   // of all but the producers, which start on K at once
        tc::fence_before_sync();
        asm volatile("barrier.cta.sync.aligned 3, %0;" ::"n"(C::SOFT + 32) : "memory");
        tc::fence_after_sync();
    };
    if (warp == C::MMA) {
        tc::tmem_alloc(&tmem_slot, 512);
        if (C::F32 && lane == 0) {
            s_slot = blockIdx.y * gridDim.x + blockIdx.x;
            if (claim) {
                unsigned at;
                asm volatile("mov.u32 %0, %%smid;" : "=r"(at));
                int tries = 64 * GB_MAX_SMS;
                for (at %= GB_MAX_SMS; !(s_claimed = atomicCAS(a.tickets + at, 0u, 1u) == 0u); at = (at + 1) % GB_MAX_SMS)
                    if (--tries == 0) {   // a workspace that was never zeroed, or is shared: the place stays another's
                        atomicExch(a.err, (unsigned)(-GB_ETIMEOUT));
                        break;
                    }
                __threadfence();
                s_slot = (int)at;
            } else if (s_slot >= GB_MAX_SMS) {
                s_slot = 0;   // no running sum
            }
        }
        __syncwarp();
    }

    // ---- Q rows, eight lanes a row (a thread per row would touch 32 lines at
    // a time: 22,000 cycles for fp32 at hd 128): fp16 into shared memory; fp32
    // scaled and split, the remainders into shared memory, the high parts
    // through the V stages into tensor memory (the A operand of two products of three)
    float up_inv = 1.f;   // 2^-e of this thread's row
    if (warp < C::MMA) {
        constexpr int NV = HD / 64, LD = C::F32 ? 2 : 1;           // a lane's runs of 8 columns, loads of each
        constexpr int STEP = C::SOFT / 8, U = 128 / STEP;          // rows of the block at a time, of a thread in flight
        const int la = lane & 7;
        int qo[U], ho[U];                                          // their queries (past the tile's: none) and columns
#pragma unroll
        for (int v = 0; v < U; v++) {
            const int rr = (tid >> 3) + v * STEP;
            qo[v] = rr < a.bq * a.group ? rr / a.group : 1 << 30;
            ho[v] = (kvh * a.group + rr % a.group) * HD + 8 * la;
        }
        for (int tile = 0; tile < (two ? 2 : 1); tile++) {
            uint4 w[U][NV][LD];
#pragma unroll
            for (int v = 0; v < U; v++) {
                const bool in = qo[v] < n_q - q0 - tile * a.bq;
                const A* src = static_cast<const A*>(a.q) + (size_t)(t_begin + q0 + tile * a.bq + qo[v]) * a.ldq + ho[v];
#pragma unroll
                for (int x = 0; x < NV; x++)
#pragma unroll
                    for (int z = 0; z < LD; z++)
                        w[v][x][z] = in ? ldg4(src + 64 * x + 4 * z) : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int v = 0; v < U; v++) {
                const int rr = (tid >> 3) + v * STEP;
                if constexpr (!C::F32) {
#pragma unroll
                        for (int x = 0; x < NV; x++)
                            *reinterpret_cast<uint4*>((C::QT ? vs : qs) + tile * C::QB + pp_off(rr, 8 * x + la, 128)) = w[v][x][0];
                } else {
                    float f[NV][8], mx = 0.f;
#pragma unroll
                    for (int x = 0; x < NV; x++)
#pragma unroll
                        for (int z = 0; z < 2; z++) {
                            const uint4 g = w[v][x][z];
                            f[x][4 * z] = __uint_as_float(g.x);
                            f[x][4 * z + 1] = __uint_as_float(g.y);
                            f[x][4 * z + 2] = __uint_as_float(g.z);
                            f[x][4 * z + 3] = __uint_as_float(g.w);
#pragma unroll
                            for (int k = 0; k < 4; k++) mx = fmaxf(mx, fabsf(f[x][4 * z + k]));
                        }
#pragma unroll
                    for (int o = 4; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                    const int e = tc::f16_scale_exp(__float_as_uint(mx));
                    const float up = tc::pow2f(e);
                    if (la == 0) s_row[tile][0][rr] = tc::pow2f(-e);
#pragma unroll
                    for (int x = 0; x < NV; x++) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const float y0 = f[x][2 * k] * up, y1 = f[x][2 * k + 1] * up;
                            hi[k] = pp_pack(y0, y1);
                            const float2 h2 = __half22float2(*reinterpret_cast<const __half2*>(&hi[k]));
                            lo[k] = pp_pack(y0 - h2.x, y1 - h2.y);
                        }
                        const uint32_t at = (uint32_t)(tile * C::QB) + pp_off(rr, 8 * x + la, 128);
                        *reinterpret_cast<uint4*>(vs + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        *reinterpret_cast<uint4*>(qs + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                }
            }
        }
    }
    if (warp <= C::MMA) {
        if constexpr (C::QT) {
            static_assert(2 * C::QB <= ST * C::KS * C::KB, "the high parts fit the stages of V");
            start_sync();
            if (warp < C::MMA) {
                if (rt == 0 || two) {
                    if (C::F32) up_inv = s_row[rt][0][r];
                    const uint32_t qh = tmem_slot + ((uint32_t)((warp & 3) * 32) << 16) + 128u + 64u * rt + (uint32_t)(hf * (HD / 4));
#pragma unroll
                    for (int u = 0; u < HD / 8 / TR; u += 4) {
                        uint32_t hi[16];
#pragma unroll
                        for (int v = 0; v < 4; v++) {
                            const uint4 w = *reinterpret_cast<const uint4*>(vs + rt * C::QB + pp_off(r, hf * (HD / 8 / TR) + u + v, 128));
                            hi[4 * v] = w.x;
                            hi[4 * v + 1] = w.y;
                            hi[4 * v + 2] = w.z;
                            hi[4 * v + 3] = w.w;
                        }
                        tc::tmem_st16_nowait(qh + 4 * u, hi);
                    }
                    tc::tmem_wait_st();
                }
                tc::fence_async_smem();   // V's copies come after these reads
                __syncwarp();
                if (lane == 0) mbs_arrive(qread);
            }
        }
        tc::fence_async_smem();
        start_sync();
    }
    const uint32_t tmem = warp <= C::MMA ? tmem_slot : 0u;
    bool ok = true, again = false;

    if (warp == C::MMA) {   // ---- MMA issue: the whole warp, uniform; one lane's instructions
        {
            // 512 columns are all of tensor memory: its base is 0
            const uint32_t lead = tc::elect();
            auto wait = [&](uint32_t bar, uint32_t parity) {
                if (ok) ok = __all_sync(0xffffffffu, mbs_wait(bar, parity, a.err));
            };
            constexpr uint32_t idS = tc::idesc_f16(128, NK), idO = tc::idesc_f16_bmn(128, HD);
            // descriptors are built once and moved by adding to their address field (16-byte units)
            const uint64_t qd = tc::smem_desc_sw128(tc::smem_u32(qs), 16, 1024);
            const uint64_t kd = tc::smem_desc_sw128(tc::smem_u32(ks), 16, 1024);
            const uint64_t vd = tc::smem_desc_sw128(tc::smem_u32(vs), NK * 128, 1024);
            auto scores = [&](int i, int st, int j) {   // S_i = Q_i K^T, the j-th tile's
                const uint32_t S = C::SW * i + (uint32_t)NK * (j % NS);
                const uint64_t qa = qd + (uint32_t)(i * (C::QB >> 4)), ka = kd + (uint32_t)(st * (C::KS * C::KB >> 4));
                // the small products first, so that the sums truncate at their size
                if (C::F32 || !C::QT)
#pragma unroll
                    for (int k = 0; k < HD / 16; k++)
                        tc::mma_f16_w(lead, S, qa + (uint32_t)(((k >> 2) * 128 * 128 + (k & 3) * 32) >> 4),
                                      ka + (uint32_t)(((k >> 2) * NK * 128 + (k & 3) * 32) >> 4), idS, k > 0);
                if (C::QT) {
                    const uint32_t qh = 128u + 64u * i;
#pragma unroll
                    for (int p = C::KS - 1; p >= 0; p--)
#pragma unroll
                        for (int k = 0; k < HD / 16; k++)
                            tc::mma_f16_ta_w(lead, S, qh + 8u * k, ka + (uint32_t)((p * C::KB + (k >> 2) * NK * 128 + (k & 3) * 32) >> 4),
                                           idS, C::F32 || p < C::KS - 1 || k > 0);
                }
                tc::mma_commit_w(lead, sfull + 8 * (2 * i + j % NS));
            };
            auto output = [&](int i, int st, int j) {   // O_i (+)= P_i V
                const uint32_t O = 256u + 128u * i, P = C::SW * i + (uint32_t)NK * (j % NS);
                const uint64_t va = vd + (uint32_t)(st * (C::KS * C::KB >> 4));
#pragma unroll
                for (int h2 = 0; h2 < TR; h2++) {   // as the parts of P arrive
                    wait(pfull + 8 * (2 * i + (TR == 2 ? h2 : j % NS)), (j / NS) & 1);
                    tc::fence_after_sync();
#pragma unroll
                    for (int p = 0; p < C::KS + 1; p++) {   // hi.hi, lo.hi (fp32), hi.lo
                        if (!C::F32 && p == 1) continue;
                        const uint32_t pa = P + (uint32_t)(NH * h2) + (p == 1 ? C::PLO : 0u);
#pragma unroll
                        for (int k = 0; k < NH / 16; k++)
                            tc::mma_f16_ta_w(lead, O + (p > 0 ? C::OS : 0u), pa + 8u * k,
                                             va + (uint32_t)(((p == 2) * C::KB + (h2 * (NH / 16) + k) * 2048) >> 4), idO,
                                             (C::F32 ? j % C::FLUSH : j) > 0 || h2 > 0 || p > (C::OS ? 1 : 0) || k > 0);
                    }
                }
                tc::mma_commit_w(lead, odone + 8 * i);
            };
            const int tiles[2] = {nt0, two ? nt : 0};   // key tiles of each row tile
            for (int j = 0; j < min(NS, nt); j++) {
                wait(kfull + 8 * (j % ST), (j / ST) & 1);
                tc::fence_after_sync();
                for (int i = 0; i < 2; i++)
                    if (j < tiles[i]) scores(i, j % ST, j);
                tc::mma_commit_w(lead, kfree + 8 * (j % ST));
            }
            for (int j = 0; j < nt; j++) {
                const int jn = j + NS, st = j % ST, sn = jn % ST;   // scores run NS tiles ahead
                wait(vfull + 8 * st, (j / ST) & 1);
                if (jn < nt) wait(kfull + 8 * sn, (jn / ST) & 1);
                for (int i = 0; i < 2; i++) {
                    if (j >= tiles[i]) continue;
                    output(i, st, j);
                    if (jn < tiles[i]) scores(i, sn, jn);
                    if (j + 1 == tiles[i]) tc::mma_commit_w(lead, ofull + 8 * i);
                }
                tc::mma_commit_w(lead, vfree + 8 * st);
                if (jn < nt) tc::mma_commit_w(lead, kfree + 8 * sn);
            }
        }
        __syncwarp();
    } else if (warp > C::MMA) {   // ---- K and V tiles
        const int pw = warp - C::MMA - 1;
        if (!C::Q8) {
            const int R = min(1 << c.shift, NK);         // rows of a box
            for (int j = 0; j < nt; j++) {
                const int st = j % ST, key0 = (j0 + j) * NK;
                const int valid = min(kend - key0, NK);  // keys of the tile
                const int nb = (valid + R - 1) / R;      // boxes that hold some
                const bool part = valid < NK;
                // a lane's boxes: page of box i (lanes share the work over boxes)
                const uint32_t bytes = (uint32_t)(nb * R * HD * 2);
                if (j >= ST) {
                    if (ok) ok = mbs_wait(kfree + 8 * st, ((j / ST) - 1) & 1, a.err);
                }
                if (lane == 0) mbs_expect(kfull + 8 * st, bytes);
                __syncwarp();
                for (int i = lane; i < nb; i += 32) {
                    const int key = key0 + i * R;
                    int page = page_of(c, b, seq, key, a.err);
                    if (page < 0) page = 0;
                    const int row = key & ((1 << c.shift) - 1);
#pragma unroll
                    for (int g = 0; g < C::G; g++)
                        tma_load_3d(tc::smem_u32(ks + st * C::KB) + g * NK * 128 + i * R * 128, &kmap, g * 64, row,
                                    page * c.n_kv + kvh, kfull + 8 * st);
                }
                if (j >= ST) {
                    if (ok) ok = mbs_wait(vfree + 8 * st, ((j / ST) - 1) & 1, a.err);
                } else if (C::QT && j == 0) {
                    if (ok) ok = mbs_wait(qread, 0, a.err);
                }
                const uint32_t vbar = part ? tail : vfull + 8 * st;
                if (lane == 0) mbs_expect(vbar, bytes);
                __syncwarp();
                for (int i = lane; i < nb; i += 32) {
                    const int key = key0 + i * R;
                    int page = page_of(c, b, seq, key, a.err);
                    if (page < 0) page = 0;
                    const int row = key & ((1 << c.shift) - 1);
#pragma unroll
                    for (int g = 0; g < C::G; g++)
                        tma_load_3d(tc::smem_u32(vs + st * C::KB) + g * NK * 128 + i * R * 128, &vmap, g * 64, row,
                                    page * c.n_kv + kvh, vbar);
                }
                if (part) {   // the last tile: zero the rows past the last key once the copies are in
                    if (ok) ok = mbs_wait(tail, 0, a.err);
                    for (int i = lane; i < (NK - valid) * 8 * C::G; i += 32) {
                        const int g = i / ((NK - valid) * 8), e = i % ((NK - valid) * 8);
                        *reinterpret_cast<uint4*>(vs + st * C::KB + g * NK * 128 + valid * 128 + e * 16) =
                            make_uint4(0u, 0u, 0u, 0u);
                    }
                    tc::fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbs_arrive(vfull + 8 * st);
                }
            }
        } else {
            // a thread: row (key) rr of the tile and 16-column runs u0 .., four at
            // a time; the next four are loaded before these are converted
            constexpr int TPR = C::Q8 ? C::PROD * 32 / NK : 1;   // threads per row
            constexpr int SUB = HD / 64 / TPR > 0 ? HD / 64 / TPR : 1;   // groups of four runs per thread and tile
            constexpr int NU = HD / 16 / TPR / SUB;      // runs of a group (two at hd 64 with two threads per row)
            const int pt = pw * 32 + lane, rr = pt % NK, u0 = (pt / NK) * SUB * NU;
            auto place = [&](int j) {                    // the row's place in a pool; none: -1
                const int key = (j0 + j) * NK + rr;
                if (j >= nt || key >= kend) return (long long)-1;
                int page = page_of(c, b, seq, key, a.err);
                if (page < 0) page = 0;
                return (long long)((size_t)page * c.page_bytes + (size_t)kvh * c.slab) +
                       (long long)(key & ((1 << c.shift) - 1)) * HD;
            };
            struct Runs {
                uint4 w[NU];
                uint32_t d;
            };
            auto load = [&](long long at, int j, int kv, int sub, Runs& o) {
#pragma unroll
                for (int i = 0; i < NU; i++) o.w[i] = make_uint4(0u, 0u, 0u, 0u);
                o.d = 0u;
                if (at >= 0) {
                    const uint8_t* pool = kv ? c.v : c.k;
                    const int u = u0 + sub * NU, row = ((j0 + j) * NK + rr) & ((1 << c.shift) - 1);
#pragma unroll
                    for (int i = 0; i < NU; i++) o.w[i] = ldg4(pool + at + (u + i) * 16);
                    const uint8_t* sp = pool + at - (long long)row * HD + ((size_t)HD << c.shift) + row * (HD / 16) + u;
                    o.d = NU == 4 ? ldg1(sp) : ldg_u16(sp);
                }
            };
            long long at = place(0), at_next = place(1);
            Runs cur, nxt;
            load(at, 0, 0, 0, cur);
            for (int j = 0; j < nt; j++) {
                const int st = j % ST;
#pragma unroll
                for (int it = 0; it < 2 * SUB; it++) {
                    const int kv = it / SUB, sub = it % SUB;
                    if (it + 1 < 2 * SUB) load(at, j, (it + 1) / SUB, (it + 1) % SUB, nxt);
                    else load(at_next, j + 1, 0, 0, nxt);
                    if (j >= ST && sub == 0) {
                        if (ok) ok = mbs_wait((kv ? vfree : kfree) + 8 * st, ((j / ST) - 1) & 1, a.err);
                    } else if (j == 0 && kv && sub == 0) {
                        if (ok) ok = mbs_wait(qread, 0, a.err);
                    }
                    uint8_t* dst = (kv ? vs : ks) + st * C::KS * C::KB;
#pragma unroll
                    for (int i = 0; i < NU; i++) {
                        const uint32_t ww[4] = {cur.w[i].x ^ 0x80808080u, cur.w[i].y ^ 0x80808080u,
                                                cur.w[i].z ^ 0x80808080u, cur.w[i].w ^ 0x80808080u};
                        uint32_t hi[8], lo[8];
                        const uint32_t dd = __byte_perm(cur.d, 0u, i / 2 ? 0x3232 : 0x1010);
                        const __half2 d2 = *reinterpret_cast<const __half2*>(&dd);
#pragma unroll
                        for (int x = 0; x < 8; x++) {   // codes as halves (1024 + 128 + code, less 1152), times the scale
                            uint32_t by = __byte_perm(ww[x >> 1], 0x64646464u, x & 1 ? 0x4342 : 0x4140);
                            const __half2 cd = __hsub2(*reinterpret_cast<__half2*>(&by), __floats2half2_rn(1152.f, 1152.f));
                            const __half2 v = __hmul2(cd, d2);
                            hi[x] = *reinterpret_cast<const uint32_t*>(&v);
                            if (C::KS == 2) {
                                const __half2 rest = __hfma2(cd, d2, __hneg2(v));
                                lo[x] = *reinterpret_cast<const uint32_t*>(&rest);
                            }
                        }
                        const int u = 2 * (u0 + sub * NU + i);
                        *reinterpret_cast<uint4*>(dst + pp_off(rr, u, NK)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        *reinterpret_cast<uint4*>(dst + pp_off(rr, u + 1, NK)) = make_uint4(hi[4], hi[5], hi[6], hi[7]);
                        if (C::KS == 2) {
                            *reinterpret_cast<uint4*>(dst + C::KB + pp_off(rr, u, NK)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                            *reinterpret_cast<uint4*>(dst + C::KB + pp_off(rr, u + 1, NK)) =
                                make_uint4(lo[4], lo[5], lo[6], lo[7]);
                        }
                    }
                    if (sub == SUB - 1) {
                        tc::fence_async_smem();
                        __syncwarp();
                        if (lane == 0) mbs_arrive((kv ? vfull : kfull) + 8 * st);
                    }
                    cur = nxt;
                }
                at = at_next;
                at_next = place(j + 2);
            }
        }
        __syncwarp();
    } else if (rt == 0 || two) {   // ---- softmax
        const uint32_t lb = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t O = lb + 256u + 128u * rt + (uint32_t)(hf * (HD / TR));
        const float sc = up_inv * (1.4426950408889634f / sqrtf((float)HD));
        const int lim = pos0 + qi;                       // the last key this row sees
        const int lim_min = pos0 + q0 + rt * a.bq;       // and the tile's first query
        const int n_tiles = rt == 0 ? nt0 : nt;          // without any O is not read
        float m = -INFINITY, l = 0.f;                    // the row's maximum, this part's sum
        // fp32: the running sum of O's columns in the workspace, [HD / 4][128 rows][4]: this CTA's partial when the keys are
        // split, else a slot of its own for as long as it runs
        float* run = a.part;
        if (C::F32) {
            run += ((size_t)s_slot * 2 + rt) * (HD + 2) * 128 + (size_t)(2 + hf * (HD / TR)) * 128 + 4 * r;
        }
        auto ld_o = [&](int c0, float (&o)[16]) {        // O's columns c0 .. + 15
            if constexpr (C::OS == 0) {
                tc::tmem_ld16(O + c0, o);
            } else {
#pragma unroll
                for (int i = 0; i < 16; i += 8) {
                    float big[8], small[8];
                    tc::tmem_ld8x2(O + c0 + i, O + C::OS + c0 + i, big, small);
#pragma unroll
                    for (int x = 0; x < 8; x++) o[i + x] = big[x] + small[x];
                }
            }
        };
        // with what the running sum holds of them
        auto read_o = [&](int c0, float (&o)[16], bool more) {
            ld_o(c0, o);
            if (C::F32 && more)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const float4 w = __ldcg(reinterpret_cast<const float4*>(run + (c0 + i) * 128));
                    o[i] += w.x;
                    o[i + 1] += w.y;
                    o[i + 2] += w.z;
                    o[i + 3] += w.w;
                }
        };
        for (int j = 0; j < n_tiles; j++) {
            const int key0 = (j0 + j) * NK, buf = j % NS;
            const uint32_t S = lb + C::SW * rt + (uint32_t)(NK * buf + NH * hf);
            const bool masked = key0 + NK - 1 > lim_min;
            const int left = (live ? lim : -1) - key0 - hf * NH;   // keys 0 .. left of the part are seen
            if (ok) ok = mbs_wait(sfull + 8 * (2 * rt + buf), (j / NS) & 1, a.err);
            tc::fence_after_sync();
            float x[NH], mx = -INFINITY;
            if (NH == 64)
                tc::tmem_ld32x2(S, S + 32, *reinterpret_cast<float (*)[32]>(x), *reinterpret_cast<float (*)[32]>(x + NH - 32));
            else
                tc::tmem_ld32(S, *reinterpret_cast<float (*)[32]>(x));
            if (masked) {
#pragma unroll
                for (int i = 0; i < NH; i++) x[i] = i <= left ? x[i] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < NH; i += 2) mx = fmaxf(mx, fmaxf(x[i], x[i + 1]));
            mx *= sc;
            auto passes = [&](float v) { return v > m + PP_TAU || (m == -INFINITY && v > -INFINITY); };
            const bool flush = C::F32 && j > 0 && j % C::FLUSH == 0;
            auto rescale = [&](float v) {   // the maximum moves to v where it passes; O with it
                const bool move = passes(v);
                const float al = !move ? 1.f : m == -INFINITY ? 0.f : pp_ex2(m - v);
                l *= al;
                m = move ? v : m;
                if (j > 0 && !flush) {
                    // P V of the tile before: with one buffer its commit came before this S; with two the
                    // commit of the one before that did, so the parity is not ambiguous
                    if (NS == 2 && ok) ok = mbs_wait(odone + 8 * rt, (j - 1) & 1, a.err);
                    tc::fence_after_sync();
#pragma unroll 1
                    for (int n = 0; n < (C::OS ? 2 : 1) * (HD / TR / 16); n++) {
                        const uint32_t at = O + (n < HD / TR / 16 ? 16u * n : C::OS + 16u * (n - HD / TR / 16));
                        float o[16];
                        tc::tmem_ld16(at, o);
#pragma unroll
                        for (int i = 0; i < 16; i++) o[i] *= al;
                        tc::tmem_st16(at, o);
                    }
                    tc::fence_before_sync();
                }
                if (C::F32 && j >= C::FLUSH && al != 1.f) {   // the running sum too
#pragma unroll 1
                    for (int c0 = 0; c0 < HD / TR; c0 += 4) {
                        float4* w = reinterpret_cast<float4*>(run + c0 * 128);
                        const float4 v = __ldcg(w);
                        __stcg(w, make_float4(v.x * al, v.y * al, v.z * al, v.w * al));
                    }
                }
            };
            auto add_up = [&] {   // what O holds (all P V before this tile) into the running sum
#pragma unroll 1
                for (int c0 = 0; c0 < HD / TR; c0 += 16) {
                    float o[16];
                    ld_o(c0, o);
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        float* to = run + (c0 + i) * 128;
                        if (j == C::FLUSH)
                            __stcg(reinterpret_cast<float4*>(to), make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]));
                        else   // its one writer
                            asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(to), "f"(o[i]), "f"(o[i + 1]),
                                         "f"(o[i + 2]), "f"(o[i + 3]) : "memory");
                    }
                }
                tc::fence_before_sync();
            };
            if (TR == 1) {
                if (__any_sync(0xffffffffu, passes(mx))) rescale(mx);
            } else if (pp_vote(1 + rt, passes(mx))) {   // of all rows of the tile
                if (flush) add_up();
                s_row[rt][hf][r] = mx;
                pp_sync(1 + rt);
                rescale(fmaxf(mx, s_row[rt][hf ^ 1][r]));
                pp_sync(1 + rt);   // O is rescaled before either part of P is handed over; s_row is free again
                tc::fence_after_sync();
            }
            else if (flush) {
                add_up();
                pp_sync(1 + rt);   // O is read before P is handed over
            }
            const float off = PP_LIFT - (m == -INFINITY ? 0.f : m);
            const float2 sc2 = make_float2(sc, sc), off2 = make_float2(off, off);
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int c0 = 0; c0 < NH; c0 += 32) {
                const float* y = x + c0;
                uint32_t ph[16], pl[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    float2 v = __ffma2_rn(make_float2(y[2 * i], y[2 * i + 1]), sc2, off2);
                    if (!C::F32 && i % PP_POLY == PP_POLY - 1) v = pp_ex2_poly(v);
                    else v = make_float2(pp_ex2(v.x), pp_ex2(v.y));
                    sum = __fadd2_rn(sum, v);
                    ph[i] = pp_pack(v.x, v.y);
                    if (C::F32) {
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&ph[i]));
                        pl[i] = pp_pack(v.x - f.x, v.y - f.y);
                    }
                }
                tc::tmem_st16_nowait(S + c0 / 2, ph);   // over the scores that this thread has read
                if (C::F32) tc::tmem_st16_nowait(S + C::PLO + c0 / 2, pl);
            }
            l += sum.x + sum.y;
            tc::tmem_wait_st();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbs_arrive(pfull + 8 * (2 * rt + (TR == 2 ? hf : buf)));
        }
        // through which the output goes: 32 rows of RB bytes, CP columns, a warp
        constexpr int WB = C::QB / (4 * TR), RB = WB / 32 < 128 ? WB / 32 : 128, UN = RB / 16;
        constexpr int CP = RB / (int)sizeof(A);
        const bool more = n_tiles > C::FLUSH;
        float4 held[C::F32 ? CP / 4 : 1];                // the running sum's, read ahead
        auto read_ahead = [&](int c1) {
            if (C::F32 && more && n_split == 1)
#pragma unroll
                for (int i = 0; i < CP / 4; i++) held[i] = __ldcg(reinterpret_cast<const float4*>(run + (c1 + 4 * i) * 128));
        };
        read_ahead(0);
        if (n_tiles > 0) {
            if (ok) ok = mbs_wait(ofull + 8 * rt, 0, a.err);
            tc::fence_after_sync();
        }
        if (TR == 2) {
            s_row[rt][hf][r] = l;
            pp_sync(1 + rt);
            l += s_row[rt][hf ^ 1][r];
        }
        if (n_split == 1) {
            // Through the row tile's part of Q, which no MMA reads any more, so
            // that a warp writes whole runs of rows.
            static_assert(CP % 16 == 0 && HD / TR % CP == 0 && (UN == 8 || UN == 4), "rows of the staging area");
            uint8_t* wb = qs + rt * C::QB + warp % (4 * TR) * WB;
            auto at = [&](int row, int u) { return wb + row * RB + ((u ^ (UN == 8 ? row & 7 : (row >> 1) & 3)) << 4); };
            // keys with scores of -inf alone: no number; no keys: the same, and zeros by pp_row
            const float inv = m == -INFINITY ? NAN : 1.0f / l;
            float odd = 0.f;                                  // no number once a result is not finite
            const unsigned long long dst = live ? reinterpret_cast<unsigned long long>(
                static_cast<A*>(a.out) + (size_t)(t_begin + qi) * a.ldo + (size_t)h * HD + hf * (HD / TR)) : 0ull;
#pragma unroll 1
            for (int c1 = 0; c1 < HD / TR; c1 += CP) {
#pragma unroll
                for (int c0 = 0; c0 < CP; c0 += 16) {
                    float o[16];
                    ld_o(c1 + c0, o);
                    if (C::F32 && more)
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const float4 w = held[C::F32 ? (c0 + i) / 4 : 0];
                            o[i] += w.x;
                            o[i + 1] += w.y;
                            o[i + 2] += w.z;
                            o[i + 3] += w.w;
                        }
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        o[i] *= inv;
                        odd = fmaf(o[i], 0.f, odd);
                    }
#pragma unroll
                    for (int i = 0; i < (int)sizeof(A); i++) {   // 16 columns: 2 or 4 units
                        const int n = 16 / (int)sizeof(A);
                        uint4 w;
                        if constexpr (C::F32) w = make_uint4(__float_as_uint(o[n * i]), __float_as_uint(o[n * i + 1]), __float_as_uint(o[n * i + 2]), __float_as_uint(o[n * i + 3]));
                        else w = make_uint4(pp_pack(o[n * i], o[n * i + 1]), pp_pack(o[n * i + 2], o[n * i + 3]), pp_pack(o[n * i + 4], o[n * i + 5]), pp_pack(o[n * i + 6], o[n * i + 7]));
                        *reinterpret_cast<uint4*>(at(lane, c0 / n + i)) = w;
                    }
                }
                if (c1 + CP < HD / TR) read_ahead(c1 + CP);
                __syncwarp();
#pragma unroll
                for (int i = 0; i < UN; i++) {
                    const int row = (i * 32 + lane) / UN, u = lane % UN;
                    const unsigned long long to = __shfl_sync(0xffffffffu, dst, row);
                    if (to) *reinterpret_cast<uint4*>(to + c1 * sizeof(A) + 16 * u) = *reinterpret_cast<const uint4*>(at(row, u));
                }
                __syncwarp();
            }
            again = live && odd != 0.f;
            if (again) atomicOr(&s_again[4 * rt + (r >> 5)], 1u << (r & 31));
        } else {   // m [128 rows], l [128], O [HD / 4][128][4] of this CTA's tile
            float* pp = a.part + (((size_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 + rt) * (HD + 2) * 128;
            if (hf == 0) {
                pp[r] = m;
                pp[128 + r] = l;
            }
            pp += (2 + hf * (HD / TR)) * 128 + 4 * r;
#pragma unroll 1
            for (int c0 = 0; c0 < HD / TR; c0 += 16) {
                float o[16];
                read_o(c0, o, more);
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *reinterpret_cast<float4*>(pp + (c0 + i) * 128) =
                        n_tiles > 0 ? make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
    }
    tc::fence_before_sync();
    again = __syncthreads_or(again);
    auto once_more = [&] {   // the noted rows, a warp each
#pragma unroll 1
        for (int i = warp; i < 256; i += C::THREADS / 32)
            if (s_again[i >> 5] >> (i & 31) & 1u) {
                const int x = i & 127, at = q0 + (i >> 7) * a.bq + x / a.group;
                pp_row<A, HD, DT>(a, seq, kvh, t_begin + at, kvh * a.group + x % a.group, pos0 + at + 1);
            }
    };
    if (warp == C::MMA) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, 512);
    }
    if (claim && tid == 0 && s_claimed) {
        __threadfence();
        atomicExch(a.tickets + s_slot, 0u);
    }
    if (n_split == 1) {
        if (again) once_more();
        return;
    }
    // ---- the last split of this row block joins them
    if (tid == 0) {
        unsigned prev;
        asm volatile("fence.acq_rel.gpu;\n\tatom.acq_rel.gpu.global.add.u32 %0, [%1], 1;"
                     : "=r"(prev)
                     : "l"(a.tickets + blockIdx.x)
                     : "memory");
        s_last = prev == (unsigned)(n_split - 1);
    }
    __syncthreads();
    if (!s_last) return;
    if (tid == 0) a.tickets[blockIdx.x] = 0u;   // every split has arrived
    if (live) {
        const size_t step = (size_t)gridDim.x * 2 * (HD + 2) * 128;   // from one split to the next
        const float* pp = a.part + ((size_t)blockIdx.x * 2 + rt) * (HD + 2) * 128 + r;
        float M = -INFINITY, L = 0.f;
        for (int z = 0; z < n_split; z++) M = fmaxf(M, __ldcg(pp + z * step));
        for (int z = 0; z < n_split; z++) {
            const float mz = __ldcg(pp + z * step);
            if (mz > -INFINITY) L = fmaf(__ldcg(pp + z * step + 128), pp_ex2(mz - M), L);
        }
        float odd = 0.f;
        const float inv = 1.0f / L;
        A* dst = static_cast<A*>(a.out) + (size_t)(t_begin + qi) * a.ldo + (size_t)h * HD;
#pragma unroll 1
        for (int c0 = hf * (HD / TR); c0 < (hf + 1) * (HD / TR); c0 += 8) {
            float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            for (int z = 0; z < n_split; z++) {
                const float mz = __ldcg(pp + z * step);
                const float f = mz > -INFINITY ? pp_ex2(mz - M) * inv : 0.f;
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    const float4 w = __ldcg(reinterpret_cast<const float4*>(pp + 3 * r + z * step + (2 + c0 + i) * 128));
                    v[i] = fmaf(f, w.x, v[i]);
                    v[i + 1] = fmaf(f, w.y, v[i + 1]);
                    v[i + 2] = fmaf(f, w.z, v[i + 2]);
                    v[i + 3] = fmaf(f, w.w, v[i + 3]);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                v[i] = M == -INFINITY ? NAN : v[i];
                odd = fmaf(v[i], 0.f, odd);
            }
            act_store8(dst + c0, v);
        }
        again = odd != 0.f;
        if (again) atomicOr(&s_again[4 * rt + (r >> 5)], 1u << (r & 31));
    }
    if (__syncthreads_or(again)) once_more();
}

template <typename A, int HD, int DT>
static int launch_prefill(const gb_kv_cache* cache, PpArgs& a, void* ws, cudaStream_t st) {
    using C = PpCfg<A, HD, DT>;
    CUtensorMap km = {}, vm = {};
    if (!C::Q8) {
        const int R = cache->page_size < C::NK ? cache->page_size : C::NK;
        if (!paged_encode(&km, cache->k, HD, cache->page_size, (size_t)cache->n_pages * a.c.n_kv, R) ||
            !paged_encode(&vm, cache->v, HD, cache->page_size, (size_t)cache->n_pages * a.c.n_kv, R))
            return GB_ECUDA;
    }
    const void* f = reinterpret_cast<const void*>(k_paged_prefill<A, HD, DT>);
    if (set_smem_once(f, C::SMEM) != cudaSuccess) return GB_ECUDA;
    // query blocks at most: the lengths are on the device
    long long blocks = a.b.cu ? (long long)a.b.n_tokens / (2 * a.bq) + a.b.n_seq : a.b.n_seq;
    if (blocks > a.b.n_tokens) blocks = a.b.n_tokens;
    const long long grid = blocks * a.c.n_kv;
    if (grid > 0x7fffffffLL) return GB_ELIMIT;
    // fewer CTAs than half the SMs: cut the keys too
    const int sms = sm_count();
    long long split = sms / grid;
    const long long most = ((long long)a.b.cap + PP_SPLIT * C::NK - 1) / (PP_SPLIT * C::NK);
    if (split > most) split = most;
    if (split < 1) split = 1;
    a.part = static_cast<float*>(ws);
    a.tickets = reinterpret_cast<unsigned*>(static_cast<uint8_t*>(ws) + PAGED_PART_BYTES);
    return launch_pdl(k_paged_prefill<A, HD, DT>, dim3((unsigned)grid, (unsigned)split), C::THREADS, C::SMEM, st, km, vm,
                      a) == cudaSuccess
               ? GB_OK
               : GB_ECUDA;
}

int paged_prefill(const gb_kv_cache* cache, const PagedView& c, const BatchView& b, int dtype, const void* q, int ldq,
                  int n_heads, void* out, int ldo, void* ws, unsigned* err, cudaStream_t st) {
    PpArgs a;
    a.c = c;
    a.b = b;
    a.q = q;
    a.out = out;
    a.ldq = ldq;
    a.ldo = ldo;
    a.group = n_heads / c.n_kv;
    a.bq = 128 / a.group;
    a.err = err;
    const int hd = cache->head_dim;
#define GB_PREFILL(T, A, HD, DT) \
    if (dtype == T && hd == HD && cache->dtype == DT) return launch_prefill<A, HD, DT>(cache, a, ws, st);
    GB_PREFILL(GB_DT_F32, float, 128, GB_DT_F16) GB_PREFILL(GB_DT_F32, float, 128, GB_DT_Q8_0)
    GB_PREFILL(GB_DT_F32, float, 64, GB_DT_F16) GB_PREFILL(GB_DT_F32, float, 64, GB_DT_Q8_0)
    GB_PREFILL(GB_DT_F16, __half, 128, GB_DT_F16) GB_PREFILL(GB_DT_F16, __half, 128, GB_DT_Q8_0)
    GB_PREFILL(GB_DT_F16, __half, 64, GB_DT_F16) GB_PREFILL(GB_DT_F16, __half, 64, GB_DT_Q8_0)
#undef GB_PREFILL
    return GB_EINVAL;
}

}  // namespace gb
