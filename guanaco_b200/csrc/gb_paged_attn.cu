// gb_paged_attn.cu -- attention over the paged KV cache: single new tokens
// (gb_paged_attention_decode) and packed prompts (gb_paged_attention_prefill).
//
//   out[t][h] = sum_p softmax_p(q[t][h] . k[p] / sqrt(hd)) v[p],  p <= position of t
//
// This file: the single-token kernel and both entry points; the prompts' kernel
// is gb_paged_prefill.cu.
#include "gb_mt.cuh"
#include "gb_paged.cuh"
#include "gb_tc.cuh"

#include <cuda.h>

#include <type_traits>

namespace gb {

// ---------------------------------------------------------------- single tokens
// S^T = K Q^T and O^T = V^T P^T on mma.sync m16n8k16 (fp16 operands, fp32
// sums): keys, then output columns, are the 16 rows, the 8 query heads of one
// KV head the 8 columns.  fp32 precision: q and the probabilities are split
// into an fp16 value and an fp16 remainder, a product each.  K and V enter
// exactly: halves as they are, Q8_0 codes as whole numbers in fp16, their
// scales applied to the sums of 32 columns (K) or to the probabilities of that
// column block (V).  The probabilities leave the first product as (key, 2
// heads) pairs and enter the second as (2 keys, head) pairs: an 8 x 8
// transposition in registers (movmatrix).
//
// The tensor cores' additions truncate, so for fp32 the products with remainders
// come first or apart and each step's P V starts from zero and is added to O
// rounded to nearest (96 sequences of up to 8066 keys, F16 cache: error against 64 bits
// 2.4e-6 -> 6.5e-7, where plain fp32 has 1.3e-6, and 271 -> 273 us; Q8_0 1.7e-6 -> 3.3e-7 (1.2e-6),
// 221 -> 235 us).
//
// Work: a step is 16 keys (Q8_0: 32, the same bytes) of one (sequence, KV
// head, 8 query heads); all
// steps of the batch, in that order, are cut into one equal run per CTA
// whatever the sequences' lengths, and the CTA's warps take its steps in turn.
// Few triples (at most half as many as CTAs): a CTA takes a piece of one, all
// pieces of one size, so that none crosses into a second triple (another
// meeting: one sequence of 8193 positions in Q8_0 21 us by runs).
// Each warp streams its own steps through a ring of TMA copies (16 rows of K and
// of V, 128- or 64-byte swizzle) and keeps its own (m, l, O); they meet once per
// segment (the steps of one such triple in this CTA) in shared memory.  A segment cut by CTA borders leaves a
// partial per CTA; the last of them to arrive joins them in CTA order.
//
// The running maximum m moves only when a score exceeds it by more than
// PD_TAU (log2 units), so a step needs no reduction but one vote; p = 2^(x - m
// + PD_LIFT) keeps the fp16 parts of small probabilities normal.  Q8_0: p
// times a scale is brought below 2^14 by a power of two, 2^-E, shared by the
// warp; l and O are in units of 2^E.
//
// 96 sequences of up to 8066 keys, 32 / 8 heads of 128, in a CUDA graph: F16 cache, fp16
// 264 us, 6360 GB/s, fp32 271 us, 6200 GB/s, bound by HBM; Q8_0, fp16 180 us, 4970
// GB/s (190 us a call among others), fp32 235 us, 3800 GB/s: some 480
// instructions per 16 keys and 8 heads, most of them turning codes into
// fragments, at the 12 warps an SM that O's and q's registers leave, issue
// 59 % of the cycles and leave HBM at 58 % (fp32 also spills 192 bytes).  One
// sequence of 8193, fp32, F16 cache: 13.7 us, latency.
constexpr int PD_W = 4;              // warps
constexpr int PD_MAX_CTAS = 4;       // CTAs per SM the workspace has room for
constexpr int PD_MC = 16;            // partials of a join in flight, and of a group
constexpr int PD_GROUP_TICKETS = GB_MAX_SMS * PD_MAX_CTAS * 2;   // two per CTA, before the segments' tickets
constexpr int PD_HEADS = 8;          // query heads of a segment
constexpr float PD_TAU = 8.f, PD_LIFT = 6.f;

template <int HD, int DT>
struct PdCfg {
    static constexpr bool Q8 = DT == GB_DT_Q8_0;
    static constexpr int KEYS = Q8 ? 32 : 16;           // keys of a step
    static constexpr int SUB = KEYS / 16;               // its runs of 16, a TMA box each
    static constexpr int SHIFT = Q8 ? 5 : 4;
    static constexpr int KB = KEYS * HD * (Q8 ? 1 : 2); // bytes of a step's K (or V) rows
    static constexpr int SB = Q8 ? KEYS * HD / 16 : 0;  // and of their scales
    static constexpr int NST = Q8 && HD == 128 ? 2 : 3; // stages: three CTAs an SM at Q8_0 and hd 128
    static constexpr int OP = HD + 4;                   // row pitch of the meeting area (bank spread)
    // shared: rows [PD_W][NST][2 KB], scales [PD_W][NST][2 SB], barriers
    // [PD_W][NST], scan [PD_W], start [4], last, free slot [PD_W].  The warps
    // meet in their rings: a warp's slot before the current one is free then,
    // and takes its O [8][OP] and (m, l) [8].
    static constexpr int SCALES = PD_W * NST * 2 * KB;
    static constexpr int BARS = SCALES + PD_W * NST * 2 * SB;
    static constexpr int SCAN = BARS + PD_W * NST * 8;
    static_assert(PD_HEADS * (OP * 4 + 8) <= 2 * KB, "a slot holds a warp's results");
    static constexpr int SMEM = SCAN + (2 * PD_W + 5) * 4;
};

// CTAs per SM: what the shared memory holds, at most PD_MAX_CTAS (registers follow).
template <int HD, int DT>
constexpr int pd_ctas() {
    return (228 * 1024) / (PdCfg<HD, DT>::SMEM + 1024) < PD_MAX_CTAS ? (228 * 1024) / (PdCfg<HD, DT>::SMEM + 1024)
                                                                     : PD_MAX_CTAS;
}

__device__ __forceinline__ void pd_tma(uint32_t dst, const void* map, int row, int slab, bool f16, uint32_t bar) {
    if (f16)
        asm volatile(
            "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %2, %4}], [%5];"
            ::"r"(dst), "l"(map), "r"(0), "r"(row), "r"(slab), "r"(bar)
            : "memory");
    else
        tma_load_3d(dst, map, 0, row, slab, bar);
}
__device__ __forceinline__ void pd_bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
// Cache row (of 8) that stands at the MMA's row n.  The swizzle spreads a
// column over the banks by the row's bits; with this order the rows that the
// lanes of one access phase read, for K (rows n) and for V (even n, odd n), all
// differ in the bits that matter.
template <int HD, int DT>
__device__ __forceinline__ int pd_row(int n) {
    if (DT == GB_DT_F16) return n ^ ((n & 1) << 2);                       // 0 5 2 7 4 1 6 3
    if (HD == 128) return n < 4 ? 2 * n : 2 * ((n & 3) ^ 1) + 1;          // 0 2 4 6 3 1 7 5
    const int h = (n & 3) ^ (n >> 2);                                     // 0 1 4 5 3 2 7 6
    return (h & 1) | (h >> 1) << 2 | (n >> 2) << 1;
}
__device__ __forceinline__ void pd_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// x, y as fp16 pairs: the rounded values and what the rounding left.
__device__ __forceinline__ void pd_split(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 r = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&r);
}
// o += A b.  fp32: with b's remainders first, from zero and then added rounded
// to nearest, as the tensor cores' additions truncate.
template <typename A>
__device__ __forceinline__ void pd_add(float (&o)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint32_t (&bh)[2],
                                       const uint32_t (&bl)[2]) {
    if (sizeof(A) == 2) {
        pd_mma(o, a0, a1, a2, a3, bh[0], bh[1]);
        return;
    }
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    pd_mma(s, a0, a1, a2, a3, bl[0], bl[1]);
    pd_mma(s, a0, a1, a2, a3, bh[0], bh[1]);
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] += s[i];
}
// A pair of values as operands: split for fp32 activations; for fp16 ones
// rounded to fp16 without a remainder (q is fp16 already; for a probability
// the error is of the size of the output's own rounding, 2.7e-4 against
// 2.1e-4 of the 64-bit result together).
template <typename A>
__device__ __forceinline__ void pd_pair(float x, float y, uint32_t& hi, uint32_t& lo) {
    if (sizeof(A) == 4) {
        pd_split(x, y, hi, lo);
    } else {
        const __half2 h = __floats2half2_rn(x, y);
        hi = *reinterpret_cast<const uint32_t*>(&h);
        lo = 0u;
    }
}
__device__ __forceinline__ uint32_t pd_transpose(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
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

// A walk over steps: sequence s, segment h of it, step st of nst; kvh: the
// segment's KV head.
template <int SHIFT>
struct PdWalk {
    int s, h, st, nst, kvh;
    __device__ __forceinline__ void go(int by, const BatchView& b, int H, int n_hg, unsigned* err) {
        st += by;
        if (st < nst) return;
        do {
            st -= nst;
            if (++h == H) {
                h = 0;
                do nst = ++s < b.n_seq ? (seq_len(b, s, err) + (1 << SHIFT) - 1) >> SHIFT : 0x7fffffff;   // past the end: no step is taken
                while (nst == 0);
            }
        } while (st >= nst);
        kvh = h / n_hg;
    }
};

// Column of position p (fragment order) of an output row.
template <int HD, int DT>
__device__ __forceinline__ int pd_col(int p) {
    const int n = p >> 3, j = p & 7;   // tile, column in the tile
    return DT == GB_DT_F16 ? (n >> 3) * 64 + 8 * j + (n & 7) : (n >> 2) * 32 + 4 * j + (n & 3);
}

template <typename A, int HD, int DT>
__global__ void __launch_bounds__(PD_W * 32, (pd_ctas<HD, DT>()))
k_paged_decode(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const PagedView c, const BatchView b, const A* __restrict__ q, int ldq, int group, int n_hg,
               A* __restrict__ out, int ldo, unsigned* __restrict__ tickets, float* __restrict__ part, unsigned* err) {
    using C = PdCfg<HD, DT>;
    constexpr int NT = HD / 8;   // output tiles of 8 columns
    constexpr int NB = HD / 32;  // 32-column blocks
    extern __shared__ __align__(1024) uint8_t sm[];   // no static shared memory: the ring starts 1024-byte aligned
    unsigned* s_scan = reinterpret_cast<unsigned*>(sm + C::SCAN);
    int* s_start = reinterpret_cast<int*>(s_scan + PD_W);
    unsigned& s_last = s_scan[PD_W + 4];
    unsigned* s_free = s_scan + PD_W + 5;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int H = c.n_kv * n_hg;
    const uint32_t bars = (uint32_t)__cvta_generic_to_shared(sm + C::BARS) + warp * C::NST * 8;
    if (lane == 0) {
        for (int i = 0; i < C::NST; i++) mbs_init(bars + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    griddep_wait();   // launched ahead of the kernel before it: nothing of it is read above

    // ---- the batch's steps and this CTA's run of them (steps < 2^31: checked on the host)
    const int per = (b.n_seq + PD_W * 32 - 1) / (PD_W * 32);
    const int s_lo = min(tid * per, b.n_seq), s_hi = min(s_lo + per, b.n_seq);
    unsigned mine = 0, live = 0;   // steps and sequences with any
    for (int s = s_lo; s < s_hi; s++) {
        const unsigned n = (seq_len(b, s, err) + C::KEYS - 1) >> C::SHIFT;
        mine += n;
        live += n > 0;
    }
    // running sums over the block's threads; total: of all
    auto scan = [&](unsigned v, unsigned& total) {
        unsigned incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) s_scan[warp] = incl;
        __syncthreads();
        total = 0;
#pragma unroll
        for (int w = 0; w < PD_W; w++) {
            if (w < warp) incl += s_scan[w];
            total += s_scan[w];
        }
        return incl;
    };
    unsigned T, n_seg;
    const unsigned incl = scan(mine, T);
    T *= H;
    __syncthreads();   // s_scan is free again
    scan(live, n_seg);
    n_seg *= H;
    // sequences without keys: zeros
    for (int s = blockIdx.x; s < b.n_seq; s += gridDim.x)
        if (seq_len(b, s, err) == 0)
            for (int i = tid; i < c.n_kv * group * HD; i += PD_W * 32) out[(size_t)s * ldo + i] = (A)0.f;
    if (T == 0) return;
    const bool pieces = 2 * n_seg <= gridDim.x;
    // steps of a CTA: a piece (a multiple of the warps; at most T / run + n_seg of them) or a run
    const unsigned run = pieces ? ((T + gridDim.x - n_seg - 1) / (gridDim.x - n_seg) + PD_W - 1) / PD_W * PD_W
                                : (T + gridDim.x - 1) / gridDim.x;
    unsigned a0 = 0, a1 = 0;   // run: this CTA's steps a0 .. a1 - 1
    if (pieces) {
        unsigned count = 0, all;
        for (int s = s_lo; s < s_hi; s++)
            count += (((seq_len(b, s, err) + C::KEYS - 1) >> C::SHIFT) + run - 1) / run * H;
        __syncthreads();
        unsigned at = scan(count, all) - count;   // first piece of sequence s_lo
        if (blockIdx.x >= all) return;
        for (int s = s_lo; s < s_hi; s++) {
            const unsigned n = (unsigned)(seq_len(b, s, err) + C::KEYS - 1) >> C::SHIFT, per_seg = (n + run - 1) / run;
            if (blockIdx.x >= at && blockIdx.x < at + per_seg * H) {
                const unsigned h = (blockIdx.x - at) / per_seg, piece = (blockIdx.x - at) % per_seg;
                s_start[0] = s;
                s_start[1] = (int)h;
                s_start[2] = (int)(piece * run);
                s_start[3] = (int)n;
            }
            at += per_seg * H;
        }
        __syncthreads();
        a1 = min(run, (unsigned)(s_start[3] - s_start[2]));
    } else {
        a0 = blockIdx.x * run;
        a1 = min(a0 + run, T);
        if (a0 >= T) return;
        unsigned at = (incl - mine) * H;   // first step of sequence s_lo
        for (int s = s_lo; s < s_hi; s++) {
            const unsigned n = (unsigned)(seq_len(b, s, err) + C::KEYS - 1) >> C::SHIFT, next = at + n * H;
            if (a0 >= at && a0 < next) {
                s_start[0] = s;
                s_start[1] = (int)((a0 - at) / n);
                s_start[2] = (int)((a0 - at) % n);
                s_start[3] = (int)n;
            }
            at = next;
        }
        __syncthreads();
    }
    const int total = (int)(a1 - a0);
    using Walk = PdWalk<C::SHIFT>;
    Walk seg = {s_start[0], s_start[1], s_start[2], s_start[3], s_start[1] / n_hg};
    Walk iss = seg;
    int iss_i = warp;   // local index of the next step to issue
    iss.go(warp, b, H, n_hg, err);

    // q of head g: columns 32 j + 8 t .. + 7
    float qx[NB][8];
    auto load_q = [&](const Walk& w) {
        const int kvh = w.kvh, hg = w.h - w.kvh * n_hg;
        const A* src = q + (size_t)w.s * ldq + (size_t)(kvh * group + hg * PD_HEADS + g) * HD + 8 * t;
#pragma unroll
        for (int j = 0; j < NB; j++) {
#pragma unroll
            for (int i = 0; i < 8; i++) qx[j][i] = 0.f;
            if (g < group - hg * PD_HEADS) act_load8(src + 32 * j, qx[j]);
        }
    };
    load_q(seg);

    uint8_t* ring_p = sm + warp * C::NST * 2 * C::KB;
    uint8_t* scales_p = sm + C::SCALES + warp * C::NST * 2 * C::SB;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(ring_p), scales = (uint32_t)__cvta_generic_to_shared(scales_p);

    // lane i < SUB sees to the step's keys 16 i .. + 15: page, box, scales
    int iss_page = 0, iss_n = 0;   // page of this lane's run; runs with keys of the sequence
    auto fetch_page = [&] {
        if (iss_i < total) {
            iss_n = C::SUB == 1 ? 1 : min(C::SUB, (seq_len(b, iss.s, err) - (iss.st << C::SHIFT) + 15) >> 4);
            iss_page = page_of(c, b, iss.s, (iss.st << C::SHIFT) + (C::SUB == 1 ? 0 : 16 * min(lane, iss_n - 1)), err);
            if (iss_page < 0) iss_page = 0;
        }
    };
    fetch_page();
    auto issue = [&](int slot) {   // every lane is done with the slot's rows
        if (iss_i >= total) return;
        const uint32_t bar = bars + 8 * slot;
        if (lane == 0) mbs_expect(bar, iss_n * (2 * (C::KB + C::SB) / C::SUB));
        __syncwarp();
        if (lane < iss_n) {
            const int row = ((iss.st << C::SHIFT) + 16 * lane) & ((1 << c.shift) - 1);
            const uint32_t dst = ring + slot * 2 * C::KB + lane * (C::KB / C::SUB);
            pd_tma(dst, &kmap, row, iss_page * c.n_kv + iss.kvh, !C::Q8, bar);
            pd_tma(dst + C::KB, &vmap, row, iss_page * c.n_kv + iss.kvh, !C::Q8, bar);
            if (C::Q8) {
                const size_t off = (size_t)iss_page * c.page_bytes + (size_t)iss.kvh * c.slab + ((size_t)HD << c.shift) +
                                   (size_t)row * (HD / 16);
                const uint32_t sdst = scales + slot * 2 * C::SB + lane * HD;
                pd_bulk(sdst, c.k + off, HD, bar);
                pd_bulk(sdst + C::SB, c.v + off, HD, bar);
            }
        }
        iss_i += PD_W;
        iss.go(PD_W, b, H, n_hg, err);
        fetch_page();
    };
#pragma unroll
    for (int i = 0; i < C::NST - 1; i++) issue(i);
    int slot = 0;
    uint32_t parity = 0;
    bool ok = true;

    // This lane's places in a step's rows; the column block j only flips bits of
    // the swizzled offset, and rows 8 on are a constant further.
    auto unit = [](int r, int u) {   // 16-byte unit u of row r
        if (!C::Q8 || HD == 128) return r * 128 + (((u ^ r) & 7) << 4);
        return r * 64 + (((u ^ (r >> 1)) & 3) << 4);
    };
    const int k_off = C::Q8 ? unit(pd_row<HD, DT>(g), t >> 1) + (t & 1) * 8 : unit(pd_row<HD, DT>(g), t);
    int v_off[2];
#pragma unroll
    for (int i = 0; i < 2; i++)
        v_off[i] = C::Q8 ? unit(pd_row<HD, DT>(2 * t + i), g >> 2) + (g & 3) * 4 : unit(pd_row<HD, DT>(2 * t + i), g);

    const float scale2 = (1.0f / sqrtf((float)HD)) * 1.4426950408889634f;
    int done = 0;            // local index where the segment starts
    int next = warp;         // local index of this warp's next step
    while (done < total) {
        const int seg_n = min(seg.nst - seg.st, total - done);   // steps of this segment here
        const int kvh = seg.kvh, hg = seg.h - seg.kvh * n_hg;
        const int n_heads = min(PD_HEADS, group - hg * PD_HEADS);
        const int len = seq_len(b, seg.s, err);
        // state of heads 2 t, 2 t + 1; O: tile pair u's columns 16 u + g, 16 u + 8 + g (fragment order)
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, thr[2] = {-INFINITY, -INFINITY}, off[2] = {0.f, 0.f}, O[NT / 2][4];
        int E = -40;
        __half top = __float2half_rn(0.f);   // 2^E, the scales' bound (0 before the first step)
#pragma unroll
        for (int n = 0; n < NT / 2; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) O[n][i] = 0.f;
        if (next < done + seg_n) {
            // ---- q scaled by a power of two per head, and split
            uint32_t qh[2 * NB][2], ql[2 * NB][2];
            float sc[2], isc[2];   // raw score -> log2 units of heads 2 t, 2 t + 1, and back
            {
                float mx = 0.f;
#pragma unroll
                for (int j = 0; j < NB; j++)
#pragma unroll
                    for (int i = 0; i < 8; i++) mx = fmaxf(mx, fabsf(qx[j][i]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const int e = tc::f16_scale_exp(__float_as_uint(mx));
                const float up = tc::pow2f(e);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int eh = __shfl_sync(0xffffffffu, e, 4 * (2 * t + i));
                    sc[i] = scale2 * tc::pow2f(-eh);
                    isc[i] = (1.0f / scale2) * tc::pow2f(eh);
                }
#pragma unroll
                for (int j = 0; j < NB; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        pd_pair<A>(qx[j][2 * i] * up, qx[j][2 * i + 1] * up, qh[2 * j + (i >> 1)][i & 1],
                                   ql[2 * j + (i >> 1)][i & 1]);
            }
            // One step; TAIL: only `left` of its keys belong to the sequence.
            auto step = [&](const uint8_t* st, const uint8_t* ss, auto tail, int left) {
                constexpr bool TAIL = decltype(tail)::value;
                const int rg = pd_row<HD, DT>(g);   // keys rg, rg + 8 stand at rows g, g + 8
                // ---- raw scores x[i][h] of keys rg + 8 i, heads 2 t + h
                float x[2 * C::SUB][2];
                if (!C::Q8) {
                    float sa[4] = {0.f, 0.f, 0.f, 0.f}, sl[4] = {0.f, 0.f, 0.f, 0.f};   // sl: with q's remainders
#pragma unroll
                    for (int j = 0; j < NB; j++) {
                        const uint8_t* kp = st + (j >> 1) * 2048 + (k_off ^ ((j & 1) * 64));
                        const uint4 k0 = *reinterpret_cast<const uint4*>(kp);
                        const uint4 k1 = *reinterpret_cast<const uint4*>(kp + 8 * 128);
                        pd_mma(sa, k0.x, k1.x, k0.y, k1.y, qh[2 * j][0], qh[2 * j][1]);
                        pd_mma(sa, k0.z, k1.z, k0.w, k1.w, qh[2 * j + 1][0], qh[2 * j + 1][1]);
                        if (sizeof(A) == 4) {
                            pd_mma(sl, k0.x, k1.x, k0.y, k1.y, ql[2 * j][0], ql[2 * j][1]);
                            pd_mma(sl, k0.z, k1.z, k0.w, k1.w, ql[2 * j + 1][0], ql[2 * j + 1][1]);
                        }
                    }
                    // an infinite score stands: the remainder of q may have the other sign than q
                    if (sizeof(A) == 4)
#pragma unroll
                        for (int i = 0; i < 4; i++) sa[i] = fabsf(sa[i]) == INFINITY ? sa[i] : sa[i] + sl[i];
                    x[0][0] = sa[0]; x[0][1] = sa[1]; x[1][0] = sa[2]; x[1][1] = sa[3];
                } else {
#pragma unroll
                    for (int u = 0; u < C::SUB; u++) {
                        __half sk[2][NB];
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            x[2 * u + i][0] = x[2 * u + i][1] = 0.f;
                            const uint8_t* sp = ss + (16 * u + 8 * i + rg) * (HD / 16);
                            if (HD == 128) *reinterpret_cast<uint2*>(&sk[i][0]) = *reinterpret_cast<const uint2*>(sp);
                            else *reinterpret_cast<uint32_t*>(&sk[i][0]) = *reinterpret_cast<const uint32_t*>(sp);
                        }
#pragma unroll
                        for (int j = 0; j < NB; j++) {
                            const uint8_t* kp = st + u * 16 * HD + (k_off ^ (j * 32));
                            uint2 w0 = *reinterpret_cast<const uint2*>(kp), w1 = *reinterpret_cast<const uint2*>(kp + 8 * HD);
                            w0.x ^= 0x80808080u; w0.y ^= 0x80808080u; w1.x ^= 0x80808080u; w1.y ^= 0x80808080u;
                            const uint32_t a0 = pd_codes(w0.x, 0x4140), a1 = pd_codes(w1.x, 0x4140);
                            const uint32_t a2 = pd_codes(w0.x, 0x4342), a3 = pd_codes(w1.x, 0x4342);
                            const uint32_t c0 = pd_codes(w0.y, 0x4140), c1 = pd_codes(w1.y, 0x4140);
                            const uint32_t c2 = pd_codes(w0.y, 0x4342), c3 = pd_codes(w1.y, 0x4342);
                            float sa[4] = {0.f, 0.f, 0.f, 0.f};
                            if (sizeof(A) == 4) {   // the small products first
                                pd_mma(sa, a0, a1, a2, a3, ql[2 * j][0], ql[2 * j][1]);
                                pd_mma(sa, c0, c1, c2, c3, ql[2 * j + 1][0], ql[2 * j + 1][1]);
                            }
                            pd_mma(sa, a0, a1, a2, a3, qh[2 * j][0], qh[2 * j][1]);
                            pd_mma(sa, c0, c1, c2, c3, qh[2 * j + 1][0], qh[2 * j + 1][1]);
                            const float d0 = __half2float(sk[0][j]), d1 = __half2float(sk[1][j]);
                            x[2 * u][0] = fmaf(sa[0], d0, x[2 * u][0]);
                            x[2 * u][1] = fmaf(sa[1], d0, x[2 * u][1]);
                            x[2 * u + 1][0] = fmaf(sa[2], d1, x[2 * u + 1][0]);
                            x[2 * u + 1][1] = fmaf(sa[3], d1, x[2 * u + 1][1]);
                        }
                    }
                }
                // ---- the V scales of keys rg + 8 i; keys past the sequence weigh nothing
                __half sv[2 * C::SUB][NB];
                if (C::Q8) {
#pragma unroll
                    for (int i = 0; i < 2 * C::SUB; i++) {
                        const uint8_t* sp = ss + C::SB + (8 * i + rg) * (HD / 16);
                        if (HD == 128) *reinterpret_cast<uint2*>(&sv[i][0]) = *reinterpret_cast<const uint2*>(sp);
                        else *reinterpret_cast<uint32_t*>(&sv[i][0]) = *reinterpret_cast<const uint32_t*>(sp);
                    }
                }
                if (TAIL) {
#pragma unroll
                    for (int i = 0; i < 2 * C::SUB; i++)
                        if (8 * i + rg >= left) {
                            x[i][0] = x[i][1] = -INFINITY;
                            if (C::Q8)
#pragma unroll
                                for (int j = 0; j < NB; j++) sv[i][j] = __float2half_rn(0.f);
                        }
                }
                // ---- does a score pass the maximum by PD_TAU, or a scale its bound?
                float mx[2] = {x[0][0], x[0][1]};
#pragma unroll
                for (int i = 1; i < 2 * C::SUB; i++) {
                    mx[0] = fmaxf(mx[0], x[i][0]);
                    mx[1] = fmaxf(mx[1], x[i][1]);
                }
                bool moved = mx[0] > thr[0] || mx[1] > thr[1];
                __half dm = __float2half_rn(0.f);
                if (C::Q8) {
                    const __half2* d2 = reinterpret_cast<const __half2*>(&sv[0][0]);
                    __half2 y = d2[0];
#pragma unroll
                    for (int j = 1; j < NB * C::SUB; j++) y = __hmax2(y, d2[j]);
                    dm = __hmax(__low2half(y), __high2half(y));
                    moved |= __hgt(dm, top);
                }
                if (__any_sync(0xffffffffu, moved)) {
                    float up = 1.f;
                    if (C::Q8) {
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) dm = __hmax(dm, __shfl_xor_sync(0xffffffffu, dm, o));
                        const int e = (int)(__float_as_uint(__half2float(dm)) >> 23) - 126;   // dm < 2^e
                        if (e > E) {
                            up = tc::pow2f(max(E - e, -126));
                            E = e;
                            top = e > 15 ? __float2half_rn(65504.f) : __float2half_rn(tc::pow2f(e));
                        }
                    }
                    float al[2];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], o));
                        const float mn = fmaxf(m[h], mx[h] * sc[h]);
                        al[h] = m[h] == -INFINITY ? 0.f : pd_ex2(m[h] - mn) * up;
                        l[h] *= al[h];
                        m[h] = mn;
                        thr[h] = (mn + PD_TAU) * isc[h];
                        // (a head with scores of -inf alone so far, moved by another's: they weigh nothing)
                        off[h] = PD_LIFT - (mn == -INFINITY ? 0.f : mn) - (C::Q8 ? (float)E : 0.f);
                    }
#pragma unroll
                    for (int n = 0; n < NT / 2; n++) {
                        O[n][0] *= al[0]; O[n][1] *= al[1]; O[n][2] *= al[0]; O[n][3] *= al[1];
                    }
                }
                float p[2 * C::SUB][2];
#pragma unroll
                for (int i = 0; i < 2 * C::SUB; i++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        p[i][h] = pd_ex2(fmaf(x[i][h], sc[h], off[h]));
                        l[h] += p[i][h];
                    }
                // ---- O^T += V^T P^T
                if (!C::Q8) {
                    uint32_t bh[2], bl[2];
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        pd_pair<A>(p[i][0], p[i][1], bh[i], bl[i]);
                        bh[i] = pd_transpose(bh[i]);
                        if (sizeof(A) == 4) bl[i] = pd_transpose(bl[i]);
                    }
#pragma unroll
                    for (int j = 0; j < HD / 64; j++) {
                        uint32_t v[4][4];
#pragma unroll
                        for (int kk = 0; kk < 4; kk++) {
                            const uint4 w = *reinterpret_cast<const uint4*>(st + C::KB + j * 2048 + (kk >> 1) * 1024 + v_off[kk & 1]);
                            v[kk][0] = w.x;
                            v[kk][1] = w.y;
                            v[kk][2] = w.z;
                            v[kk][3] = w.w;
                            if (TAIL && pd_row<HD, DT>(2 * t + (kk & 1)) + (kk >> 1) * 8 >= left)   // stale rows may hold anything
                                v[kk][0] = v[kk][1] = v[kk][2] = v[kk][3] = 0u;
                        }
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint32_t a0 = __byte_perm(v[0][e], v[1][e], 0x5410), a1 = __byte_perm(v[0][e], v[1][e], 0x7632);
                            const uint32_t a2 = __byte_perm(v[2][e], v[3][e], 0x5410), a3 = __byte_perm(v[2][e], v[3][e], 0x7632);
                            pd_add<A>(O[j * 4 + e], a0, a1, a2, a3, bh, bl);
                        }
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < C::SUB; u++)
#pragma unroll
                        for (int j = 0; j < NB; j++) {
                            uint32_t bh[2], bl[2], w[4];
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                const float d = __half2float(sv[2 * u + i][j]);
                                pd_pair<A>(p[2 * u + i][0] * d, p[2 * u + i][1] * d, bh[i], bl[i]);
                                bh[i] = pd_transpose(bh[i]);
                                if (sizeof(A) == 4) bl[i] = pd_transpose(bl[i]);
                            }
#pragma unroll
                            for (int kk = 0; kk < 4; kk++)
                                w[kk] = *reinterpret_cast<const uint32_t*>(st + C::KB + (16 * u + (kk >> 1) * 8) * HD +
                                                                           (v_off[kk & 1] ^ (j * 32))) ^
                                        0x80808080u;
#pragma unroll
                            for (int e = 0; e < 2; e++) {   // bytes 2 e, 2 e + 1 of the keys' words
                                const uint32_t lo = __byte_perm(w[0], w[1], e ? 0x7362 : 0x5140);
                                const uint32_t hi = __byte_perm(w[2], w[3], e ? 0x7362 : 0x5140);
                                const uint32_t a0 = pd_codes(lo, 0x4140), a1 = pd_codes(lo, 0x4342);
                                const uint32_t a2 = pd_codes(hi, 0x4140), a3 = pd_codes(hi, 0x4342);
                                pd_add<A>(O[j * 2 + e], a0, a1, a2, a3, bh, bl);
                            }
                        }
                }
            };
            for (; next < done + seg_n; next += PD_W) {
                __syncwarp();   // the slot before has been read
                issue(slot == 0 ? C::NST - 1 : slot - 1);
                if (ok) ok = mbs_wait(bars + 8 * slot, parity, err);
                const uint8_t *st = ring_p + slot * 2 * C::KB, *ss = scales_p + slot * 2 * C::SB;
                if (++slot == C::NST) {
                    slot = 0;
                    parity ^= 1;
                }
                const int left = len - ((seg.st + next - done) << C::SHIFT);   // at least 1
                if (left >= C::KEYS) step(st, ss, std::false_type{}, C::KEYS);
                else step(st, ss, std::true_type{}, left);
            }
        }
        // the next segment and its q, ahead of the meeting
        Walk after = seg;
        if (done + seg_n < total) {
            after.go(seg_n, b, H, n_hg, err);
            load_q(after);
        }
        // ---- the warps meet
        {
            const float u = C::Q8 ? tc::pow2f(E) : 1.f;
            const int prev = slot == 0 ? C::NST - 1 : slot - 1;   // not issued again yet
            float* meet = reinterpret_cast<float*>(ring_p + prev * 2 * C::KB);
            if (lane == 0) s_free[warp] = (unsigned)prev;
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], o);
                if (g == 0)
                    reinterpret_cast<float2*>(meet + PD_HEADS * C::OP)[2 * t + h] = make_float2(m[h], l[h] * u);
                float* row = meet + (2 * t + h) * C::OP + g;
                if (2 * t + h < n_heads)
#pragma unroll
                    for (int n = 0; n < NT / 2; n++) {
                        row[16 * n] = O[n][h] * u;
                        row[16 * n + 8] = O[n][2 + h] * u;
                    }
            }
        }
        __syncthreads();
        // the CTAs that hold the segment: c0 .. c1; a CTA's second partial is of the segment that it begins
        unsigned c0, c1;
        if (pieces) {
            c0 = blockIdx.x - (unsigned)seg.st / run;
            c1 = c0 + ((unsigned)seg.nst + run - 1) / run - 1;
        } else {
            const unsigned gs = a0 + done - seg.st;
            c0 = gs / run;
            c1 = (gs + seg.nst - 1) / run;
        }
        const bool whole = c0 == c1;
        const unsigned second = PD_HEADS * (HD + 2);
        float* mp = part + (size_t)blockIdx.x * 2 * second + (c0 == blockIdx.x ? second : 0);
        const size_t o0 = (size_t)seg.s * ldo + (size_t)(kvh * group + hg * PD_HEADS) * HD;
        const float* meets[PD_W];
#pragma unroll
        for (int w = 0; w < PD_W; w++)
            meets[w] = reinterpret_cast<const float*>(sm + (w * C::NST + s_free[w]) * 2 * C::KB);
        for (int i = tid; i < n_heads * HD; i += PD_W * 32) {
            const int h = i / HD, p = i % HD;
            float2 ml[PD_W];
            float M = -INFINITY, L = 0.f, V = 0.f;
#pragma unroll
            for (int w = 0; w < PD_W; w++) {
                ml[w] = reinterpret_cast<const float2*>(meets[w] + PD_HEADS * C::OP)[h];
                M = fmaxf(M, ml[w].x);
            }
#pragma unroll
            for (int w = 0; w < PD_W; w++) {
                const float f = ml[w].x == -INFINITY ? 0.f : pd_ex2(ml[w].x - M);
                L = fmaf(ml[w].y, f, L);
                V = fmaf(meets[w][h * C::OP + p], f, V);   // (an infinity that weighs nothing is no number)
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
            constexpr size_t PS = PD_HEADS * (HD + 2);   // floats of a partial: (m, l) [8], O [8][HD]
            // partials in, in order, thread = four neighbouring positions of a head, PD_MC of them in
            // flight; out: a partial, or (nullptr) the output
            auto join = [&](unsigned count, auto at, float* to) {
                for (int i = 4 * tid; i < n_heads * HD; i += 4 * PD_W * 32) {
                    const int h = i / HD, p = i % HD;
                    float M = -INFINITY, L = 0.f;
                    float4 V = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (unsigned k = 0; k < count; k += PD_MC) {
                        float2 ml[PD_MC];
                        float4 v[PD_MC];
                        float mn = M;
#pragma unroll
                        for (unsigned u = 0; u < PD_MC; u++) {
                            const float* pp = at(min(k + u, count - 1));
                            ml[u] = __ldcg(reinterpret_cast<const float2*>(pp) + h);
                            v[u] = __ldcg(reinterpret_cast<const float4*>(pp + 2 * PD_HEADS + i));
                        }
#pragma unroll
                        for (unsigned u = 0; u < PD_MC; u++) {
                            if (k + u >= count) ml[u] = make_float2(-INFINITY, 0.f);
                            mn = fmaxf(mn, ml[u].x);
                        }
                        const float ref = mn == -INFINITY ? 0.f : mn;   // (partials of scores of -inf alone)
                        const float fa = pd_ex2(M - ref);   // 0 before the first partial
                        M = mn;
                        L *= fa;
                        V = make_float4(V.x * fa, V.y * fa, V.z * fa, V.w * fa);
#pragma unroll
                        for (unsigned u = 0; u < PD_MC; u++) {
                            const float f = pd_ex2(ml[u].x - ref);
                            L = fmaf(ml[u].y, f, L);
                            V = make_float4(fmaf(v[u].x, f, V.x), fmaf(v[u].y, f, V.y), fmaf(v[u].z, f, V.z),
                                            fmaf(v[u].w, f, V.w));
                        }
                    }
                    if (to) {
                        *reinterpret_cast<float4*>(to + 2 * PD_HEADS + i) = V;
                        if (p == 0) {
                            to[2 * h] = M;
                            to[2 * h + 1] = L;
                        }
                    } else {
                        const float inv = 1.0f / L, r[4] = {V.x * inv, V.y * inv, V.z * inv, V.w * inv};
#pragma unroll
                        for (int u = 0; u < 4; u++) out[o0 + (size_t)h * HD + pd_col<HD, DT>(p + u)] = (A)r[u];
                    }
                }
            };
            // this CTA's arrival; true in the last of `count`, which re-arms the ticket
            auto last_of = [&](unsigned* ticket, unsigned count) {
                __syncthreads();
                if (tid == 0) {
                    unsigned prev;
                    asm volatile("fence.acq_rel.gpu;\n\tatom.acq_rel.gpu.global.add.u32 %0, [%1], 1;"
                                 : "=r"(prev)
                                 : "l"(ticket)
                                 : "memory");
                    s_last = prev == count - 1;
                    if (s_last) *ticket = 0u;
                }
                __syncthreads();
                return s_last != 0;
            };
            const unsigned count = c1 - c0 + 1;
            unsigned* ticket = tickets + PD_GROUP_TICKETS + (size_t)seg.s * H + seg.h;
            auto partial = [&](unsigned k) { return part + (size_t)(c0 + k) * 2 * PS + (k == 0 ? PS : 0); };
            if (count <= 3 * PD_MC) {
                if (last_of(ticket, count)) join(count, partial, nullptr);
            } else {   // groups of PD_MC first: one CTA alone would read them all too slowly
                const unsigned g = (blockIdx.x - c0) / PD_MC, n_groups = (count + PD_MC - 1) / PD_MC;
                const unsigned in_group = min((unsigned)PD_MC, count - g * PD_MC);
                // a group's ticket and result stand at its first CTA, where, as with the partials, two
                // segments may meet: the one that ends there and the one that begins
                float* groups = part + (size_t)gridDim.x * 2 * PS;
                auto place = [&](unsigned k) { return (size_t)(c0 + k * PD_MC) * 2 + (k == 0); };
                auto group = [&](unsigned k) { return groups + place(k) * PS; };
                if (last_of(tickets + place(g), in_group)) {
                    join(in_group, [&](unsigned k) { return partial(g * PD_MC + k); }, group(g));
                    if (last_of(ticket, n_groups)) join(n_groups, group, nullptr);
                }
            }
        }
        tc::fence_async_smem();   // the slots go back to the copies
        __syncthreads();
        done += seg_n;
        seg = after;
    }
}

static_assert((size_t)GB_MAX_SMS * PD_MAX_CTAS * 4 * PD_HEADS * (128 + 2) * 4 <= PAGED_PART_BYTES, "workspace");

template <typename A, int HD, int DT>
static cudaError_t launch_decode(const PagedView& c, const BatchView& b, const void* q, int ldq, int group, void* out,
                                 int ldo, void* ws, unsigned* err, cudaStream_t st) {
    using C = PdCfg<HD, DT>;
    const void* f = reinterpret_cast<const void*>(k_paged_decode<A, HD, DT>);
    cudaError_t e = set_smem_once(f, C::SMEM);
    if (e != cudaSuccess) return e;
    CUtensorMap km = {}, vm = {};
    if (!paged_encode_steps(&km, c.k, DT, HD, 1 << c.shift, (size_t)c.n_pages * c.n_kv) ||
        !paged_encode_steps(&vm, c.v, DT, HD, 1 << c.shift, (size_t)c.n_pages * c.n_kv))
        return cudaErrorUnknown;
    const int n_hg = (group + PD_HEADS - 1) / PD_HEADS;
    unsigned* tickets = reinterpret_cast<unsigned*>(static_cast<uint8_t*>(ws) + PAGED_TICKETS_AT);
    return launch_pdl(k_paged_decode<A, HD, DT>, dim3(sm_count() * pd_ctas<HD, DT>()), PD_W * 32, C::SMEM, st, km, vm, c, b,
                      static_cast<const A*>(q), ldq, group, n_hg, static_cast<A*>(out), ldo, tickets,
                      static_cast<float*>(ws), err);
}

static int paged_attention(const gb_kv_cache* cache, const gb_kv_batch* batch, int dtype, const void* q, int ldq,
                           int n_heads, void* out, int ldo, void* ws, cudaStream_t st, bool decode) {
    PagedView c;
    BatchView b;
    int rc = paged_views(cache, batch, &c, &b);
    if (rc) return rc;
    if (dtype != GB_DT_F32 && dtype != GB_DT_F16) return GB_EINVAL;
    if (b.n_seq == 0 || b.n_tokens == 0) return GB_OK;   // (rows of none may be anywhere)
    const int hd = cache->head_dim;
    const long long width = (long long)n_heads * hd;
    if (n_heads <= 0 || n_heads % c.n_kv || !ws || (reinterpret_cast<uintptr_t>(ws) & 15) ||
        !paged_rows_ok(dtype, q, ldq, width) || !paged_rows_ok(dtype, out, ldo, width))
        return GB_EINVAL;
    const int group = n_heads / c.n_kv;
    const long long heads8 = (long long)c.n_kv * ((group + PD_HEADS - 1) / PD_HEADS);
    if (decode ? (double)b.n_seq * (b.cap / 16 + 1) * heads8 > 0x7fffffff   // steps
               : group > 128)                                               // rows of a query
        return GB_ELIMIT;
    unsigned* err = paged_err();
    if (!err) return GB_ECUDA;
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
    return paged_prefill(cache, c, b, dtype, q, ldq, n_heads, out, ldo, ws, err, st);
}

}  // namespace gb

using namespace gb;

extern "C" size_t gb_paged_workspace_bytes(int n_heads, int n_kv_heads, int head_dim, int n_seq) {
    if (n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads || (head_dim != 64 && head_dim != 128) || n_seq < 0)
        return 0;
    const int group = n_heads / n_kv_heads, n_hg = (group + PD_HEADS - 1) / PD_HEADS;
    return PAGED_TICKETS_AT + (((size_t)PD_GROUP_TICKETS + (size_t)n_seq * n_kv_heads * n_hg) * sizeof(unsigned) + 15) / 16 * 16;
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
