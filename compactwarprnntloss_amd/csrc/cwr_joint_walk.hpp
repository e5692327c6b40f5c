// How the output-layer kernels walk the product logits[r, v] = sum_k h[r, k] * W[v, k] + bias[v]: the two
// tilings (data rows streamed through LDS, or resident in registers) hand every finished tile of
// fp32 accumulators to their caller.  In a 32x32 block of accumulators a lane holds 16 vocabulary entries
// (acc_row) of the data row lane % 32; with SWAP it is the other way round, 16 data rows of one entry.
#pragma once

#include "cwr_device.hpp"

namespace cwr {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// streaming tiling
constexpr int kJM = 256;     // data rows per workgroup
constexpr int kJN = 128;     // vocabulary entries per tile
constexpr int kJK = 32;      // K-slice
constexpr int kJPitch = 40;  // LDS row pitch in elements: 80 bytes, so that the 16-byte reads of 16 consecutive
                             // rows fall into 16 different groups of four banks

template <typename T> struct Mfma;
template <> struct Mfma<bf16_t> {
    static __device__ __forceinline__ f32x16 mac(v4i a, v4i b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
};
template <> struct Mfma<__half> {
    static __device__ __forceinline__ f32x16 mac(v4i a, v4i b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                      0, 0, 0);
    }
};

// Vocabulary entry held by accumulator register r of a 32x32 block, relative to the block's first
// entry, for a lane of half `hf` = lane / 32 (the block's data row is lane % 32).
__device__ __forceinline__ constexpr int acc_row(int r, int hf) { return 8 * (r >> 2) + 4 * hf + (r & 3); }

// The walk of the streaming kernels: every complete tile of logits is handed to
// tile(acc, first vocabulary entry of this wave's part); acc[mv][nd] is the 32x32 block of vocabulary
// entries [32 mv, 32 mv + 32) of the wave's part and data rows [32 nd, 32 nd + 32) of its 128.
template <typename T> struct StreamLds {
    T h[2][kJM][kJPitch];
    T w[2][kJN][kJPitch];
    float bias[2][kJN];  // what the accumulators of a tile start from
};

template <typename T, typename TB, bool SWAP = false, typename TileFn>
__device__ __forceinline__ void walk_streaming(const T* __restrict__ h, const T* __restrict__ W,
                                               const TB* __restrict__ bias, i64 R, int H, int V, i64 row0,
                                               StreamLds<T>& lds, TileFn&& tile) {
    auto& s_h = lds.h;
    auto& s_w = lds.w;
    auto& s_bias = lds.bias;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wd = w & 1, wv = w >> 1;
    const int hf = lane >> 5, l32 = lane & 31;

    // ---- global -> LDS staging: thread t moves 16-byte piece (t % 4) of rows t / 4 + 64 p ----------
    // The loads of a K-slice are issued TWO slices ahead of its use (two register sets taking turns):
    // one slice of matrix work is shorter than a trip to L2.
    const int st_row = tid >> 2, st_piece = tid & 3;
    // rows beyond the tensor are multiplied like the last one and dropped
    const i64 last_row = R - 1;
    const int nk = H / kJK;
    const int nvt = (V + kJN - 1) / kJN;
    const int iters = nk * nvt;
    struct Pre { v4i h[4], w[2]; };
    Pre pre[2];

    auto fetch = [&](int it, Pre& q) {
        const int vt = it / nk, kc = it - vt * nk;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            i64 r = row0 + st_row + 64 * p;
            r = r < last_row ? r : last_row;
            q.h[p] = *reinterpret_cast<const v4i*>(h + r * (i64)H + kc * kJK + st_piece * 8);
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            int v = vt * kJN + st_row + 64 * p;
            if (v >= V) v = V - 1;  // entries beyond the vocabulary are masked in the accumulator
            q.w[p] = *reinterpret_cast<const v4i*>(W + (i64)v * H + kc * kJK + st_piece * 8);
        }
    };
    auto stage = [&](int buf, const Pre& q) {
#pragma unroll
        for (int p = 0; p < 4; ++p) *reinterpret_cast<v4i*>(&s_h[buf][st_row + 64 * p][st_piece * 8]) = q.h[p];
#pragma unroll
        for (int p = 0; p < 2; ++p) *reinterpret_cast<v4i*>(&s_w[buf][st_row + 64 * p][st_piece * 8]) = q.w[p];
    };

    // the bias of a tile (-inf beyond the vocabulary, which no finite product changes and which drops
    // out of both the maximum and the sum) is fetched by the first 128 threads one tile ahead
    auto bias_of = [&](int vt) {
        const int v = vt * kJN + tid;
        return v < V ? (bias ? Elem<TB>::to_f32(bias[v]) : 0.f) : -INFINITY;
    };
    float bias_next = 0.f;
    if (tid < kJN) s_bias[0][tid] = bias_of(0);

    f32x16 acc[2][4];
    fetch(0, pre[0]);
    if (iters > 1) fetch(1, pre[1]);
    stage(0, pre[0]);
    __syncthreads();

    // one slice: slice `it` is multiplied out of LDS buffer it & 1; the loads of slice it + 2 go out
    // into the register set that slice it's own loads came through, and slice it + 1 (loaded during
    // slice it - 1) moves from the other set into the other buffer
    auto slice = [&](const int it, Pre& mine, Pre& next) {
        const int vt = it / nk, kc = it - vt * nk;
        const int buf = it & 1;
        const int v_wave = vt * kJN + 64 * wv;  // first vocabulary entry of this wave's part of the tile
        if (kc == 0) {
#pragma unroll
            for (int mv = 0; mv < 2; ++mv)
#pragma unroll
                for (int b4 = 0; b4 < 4; ++b4) {
                    float4 bq = *reinterpret_cast<const float4*>(&s_bias[vt & 1][64 * wv + 32 * mv + 8 * b4 + 4 * hf]);
                    if (SWAP) bq.x = bq.y = bq.z = bq.w = s_bias[vt & 1][64 * wv + 32 * mv + l32];
#pragma unroll
                    for (int nd = 0; nd < 4; ++nd) {
                        acc[mv][nd][4 * b4 + 0] = bq.x; acc[mv][nd][4 * b4 + 1] = bq.y;
                        acc[mv][nd][4 * b4 + 2] = bq.z; acc[mv][nd][4 * b4 + 3] = bq.w;
                    }
                }
            if (tid < kJN && vt + 1 < nvt) bias_next = bias_of(vt + 1);
        }
        if (kc == nk - 1 && tid < kJN && vt + 1 < nvt) s_bias[(vt + 1) & 1][tid] = bias_next;  // before the barrier below
        if (it + 2 < iters) fetch(it + 2, mine);
#pragma unroll
        for (int ks = 0; ks < kJK / 16; ++ks) {
            v4i fa[2], fb[4];
#pragma unroll
            for (int mv = 0; mv < 2; ++mv)
                fa[mv] = *reinterpret_cast<const v4i*>(&s_w[buf][64 * wv + 32 * mv + l32][16 * ks + 8 * hf]);
#pragma unroll
            for (int nd = 0; nd < 4; ++nd)
                fb[nd] = *reinterpret_cast<const v4i*>(&s_h[buf][128 * wd + 32 * nd + l32][16 * ks + 8 * hf]);
#pragma unroll
            for (int mv = 0; mv < 2; ++mv)
#pragma unroll
                for (int nd = 0; nd < 4; ++nd)
                    acc[mv][nd] = SWAP ? Mfma<T>::mac(fb[nd], fa[mv], acc[mv][nd]) : Mfma<T>::mac(fa[mv], fb[nd], acc[mv][nd]);
        }
        if (it + 1 < iters) stage(buf ^ 1, next);
        __syncthreads();
        if (kc != nk - 1) return;

        tile(acc, v_wave);
    };
    for (int it = 0; it < iters; it += 2) {
        slice(it, pre[0], pre[1]);
        if (it + 1 < iters) slice(it + 1, pre[1], pre[0]);
    }

}

// ---------------------------------------------------------------------------------------------
// data rows resident in registers
// ---------------------------------------------------------------------------------------------
// The streaming kernels above read their h tile once per vocabulary tile: V / 128 times in all, from
// HBM, since the tiles of all resident workgroups together exceed the L2 (measured on N=32, V=1024,
// H=512: 3.3 GB fetched for 0.32 GB of h, and the kernel runs at the speed of that traffic).  Here
// every wave keeps the MFMA operand fragments of its OWN 32 ND data rows in registers for the whole
// kernel (ND * H / 16 registers of 16 bytes per lane: the whole K range), so h is read exactly once;
// only the weight tile travels through LDS, in K-slices of 64, and every wave multiplies its rows
// with the whole tile of 128 vocabulary entries.  Needs H known at compile time (the fragments are
// indexed statically).
// (the weight tile's K-slice RK is a parameter; its LDS rows are RK + 8 elements apart: 16 bytes past a
// multiple of 128, so that 8 consecutive rows start in 8 different groups of four banks)

// Workgroup barrier that waits for this wave's LDS traffic only, never for the global loads it has in
// flight (a __syncthreads() drains those too: the weight loads issued ahead, and at the start of
// a workgroup the loads of the resident rows).
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0); vmcnt and expcnt untouched
    __builtin_amdgcn_s_barrier();
}

template <typename T, int NMV, int RK> struct ResLds {
    T w[2][32 * NMV][RK + 8];
    float bias[2][32 * NMV];  // what the accumulators of a tile start from
};

// this wave's data rows [row0, row0 + 32 ND), as MFMA operand fragments
template <typename T, int ND, int KS /* H / 16 */>
__device__ __forceinline__ void load_resident_rows(const T* __restrict__ h, i64 R, i64 row0, v4i (&hreg)[ND][KS]) {
    const int lane = threadIdx.x & 63;
    const int hf = lane >> 5, l32 = lane & 31;
    const i64 last_row = R - 1;
#pragma unroll
    for (int nd = 0; nd < ND; ++nd) {
        i64 r = row0 + 32 * nd + l32;
        r = r < last_row ? r : last_row;  // rows beyond the tensor are multiplied like the last one and dropped
        const T* src = h + r * (i64)(KS * 16) + 8 * hf;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) hreg[nd][ks] = *reinterpret_cast<const v4i*>(src + 16 * ks);
    }
}

// tile(acc, v0) receives acc[mv][nd] = vocabulary entries [v0 + 32 mv, v0 + 32 mv + 32) x data rows
// [row0 + 32 nd, row0 + 32 nd + 32) of this wave; the vocabulary is walked in tiles of JN = 32 NMV.
// Order of the start-up, which every workgroup of a round runs at the same time as every other: the
// first weight slice is requested, then the resident rows (from HBM), then after_issue() runs
// (what the caller still has to do about its rows: loads issued here queue up BEHIND the rows',
// whatever the caller asked for earlier is served before them), and the first tile starts as
// soon as the first fragments are there.
template <typename T, int ND, int KS, int NMV, int WAVES, int RK, bool D2, bool SWAP = false, typename LoadRows,
          typename TB, typename AfterIssue, typename TileFn>
__device__ __forceinline__ void walk_resident(LoadRows&& load_rows, const T* __restrict__ W,
                                              const TB* __restrict__ bias, int V, ResLds<T, NMV, RK>& lds,
                                              AfterIssue&& after_issue, TileFn&& tile) {
    constexpr int JN = 32 * NMV;
    constexpr int H = KS * 16;
    constexpr int NK = H / RK;  // K-slices per vocabulary tile
    static_assert(H % RK == 0, "whole K-slices");
    auto& s_w = lds.w;
    auto& s_bias = lds.bias;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int hf = lane >> 5, l32 = lane & 31;

    // ---- weight tile: a row of the slice is PPR pieces of 16 bytes; thread t moves piece t % PPR of rows
    // t / PPR + RPP p ----------
    constexpr int PPR = RK / 8;
    constexpr int RPP = 64 * WAVES / PPR;  // rows the workgroup moves per pass
    constexpr int NP = JN / RPP;           // passes per K-slice
    static_assert(JN % RPP == 0, "whole passes");
    const int st_row = tid / PPR, st_piece = tid % PPR;
    struct Pre { v4i w[NP]; };
    Pre pre[D2 ? 2 : 1];
    const int nvt = (V + JN - 1) / JN;
    auto fetch = [&](int vt, int kc, Pre& q) {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            int v = vt * JN + st_row + RPP * p;
            if (v >= V) v = V - 1;  // entries beyond the vocabulary are masked in the accumulator
            q.w[p] = *reinterpret_cast<const v4i*>(W + (i64)v * H + kc * RK + st_piece * 8);
        }
    };
    auto stage = [&](int buf, const Pre& q) {
#pragma unroll
        for (int p = 0; p < NP; ++p) *reinterpret_cast<v4i*>(&s_w[buf][st_row + RPP * p][st_piece * 8]) = q.w[p];
    };

    // slices are numbered it = vt * NK + kc; slice it is multiplied out of buffer it & 1 (NK is even
    // or the parity is carried), its loads were issued two slices earlier
    // the bias of a tile (-inf beyond the vocabulary, which no finite product changes and which drops
    // out of both the maximum and the sum) is fetched by the first 128 threads one tile ahead
    auto bias_of = [&](int vt) {
        const int v = vt * JN + tid;
        return v < V ? (bias ? Elem<TB>::to_f32(bias[v]) : 0.f) : -INFINITY;
    };
    float bias_next = 0.f;
    if (tid < JN) s_bias[0][tid] = bias_of(0);
    v4i hreg[ND][KS];
    load_rows(hreg);
    after_issue();
    fetch(0, 0, pre[0]);
    if (D2 && (NK > 1 || nvt > 1)) fetch(NK > 1 ? 0 : 1, NK > 1 ? 1 : 0, pre[1]);
    stage(0, pre[0]);
    lds_barrier();

    f32x16 acc[NMV][ND];
    int par = 0;  // buffer of the current slice
    // one vocabulary tile.  The first is a copy of its own: it follows the loads of the resident rows
    // in straight-line code, so its K-steps wait for the fragments they use, one after the other,
    // instead of for all of them in front of the loop.
    auto one_tile = [&](const int vt) {
#pragma unroll
        for (int mv = 0; mv < NMV; ++mv)
#pragma unroll
            for (int b4 = 0; b4 < 4; ++b4) {
                float4 bq = *reinterpret_cast<const float4*>(&s_bias[vt & 1][32 * mv + 8 * b4 + 4 * hf]);
                if (SWAP) bq.x = bq.y = bq.z = bq.w = s_bias[vt & 1][32 * mv + l32];
#pragma unroll
                for (int nd = 0; nd < ND; ++nd) {
                    acc[mv][nd][4 * b4 + 0] = bq.x; acc[mv][nd][4 * b4 + 1] = bq.y;
                    acc[mv][nd][4 * b4 + 2] = bq.z; acc[mv][nd][4 * b4 + 3] = bq.w;
                }
            }
        if (tid < JN && vt + 1 < nvt) bias_next = bias_of(vt + 1);
#pragma unroll
        for (int kc = 0; kc < NK; ++kc) {
            if (kc == NK - 1 && tid < JN && vt + 1 < nvt) s_bias[(vt + 1) & 1][tid] = bias_next;  // before its barrier
            // register set kc & 1 held this slice's loads (already staged); it now takes slice it + 2
            if (D2) {
                const int k2 = kc + 2;
                const int vt2 = vt + k2 / NK, kc2 = k2 % NK;
                if (vt2 < nvt) fetch(vt2, kc2, pre[(kc + (NK & 1) * vt) & 1]);
            } else {
                const int k1 = kc + 1;
                const int vt1 = vt + k1 / NK, kc1 = k1 % NK;
                if (vt1 < nvt) fetch(vt1, kc1, pre[0]);
            }
            // The four weight fragments of a K-step are requested together and the matrix
            // instructions follow as they arrive (left to itself the compiler reuses ONE fragment
            // register and pays the LDS latency in front of every matrix instruction).
#pragma unroll
            for (int ks = 0; ks < RK / 16; ++ks) {
                v4i fa[NMV];
#pragma unroll
                for (int mv = 0; mv < NMV; ++mv)
                    fa[mv] = *reinterpret_cast<const v4i*>(&s_w[par][32 * mv + l32][16 * ks + 8 * hf]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int mv = 0; mv < NMV; ++mv)
#pragma unroll
                    for (int nd = 0; nd < ND; ++nd)
                        acc[mv][nd] = SWAP ? Mfma<T>::mac(hreg[nd][kc * (RK / 16) + ks], fa[mv], acc[mv][nd])
                                           : Mfma<T>::mac(fa[mv], hreg[nd][kc * (RK / 16) + ks], acc[mv][nd]);
                __builtin_amdgcn_sched_barrier(0);
            }
            {
                const int k1 = kc + 1;
                const int vt1 = vt + k1 / NK;
                if (vt1 < nvt) stage(par ^ 1, pre[D2 ? (kc + 1 + (NK & 1) * vt) & 1 : 0]);
            }
            lds_barrier();
            par ^= 1;
        }
        tile(acc, vt * JN);
    };
    one_tile(0);
    for (int vt = 1; vt < nvt; ++vt) one_tile(vt);
}

}  // namespace cwr
