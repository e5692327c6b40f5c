// What the row kernels of scores.hip and distill.hip share: a row of V logits cut into 16-byte packs,
// 16 elements per lane and chunk, and the cross-lane reductions over the lanes that share a row.
//
// A chunk is 16 G elements held by G consecutive lanes: pack i of lane l covers elements
// ((i G + l) VEC - off) .. + VEC, so that the lanes of one load instruction touch consecutive
// 16-byte packs.  `off` shifts the packs of a row that does not start on a 16-byte boundary back to
// that grid; the packs at its two ends then stick out of the row.
#pragma once

#include "cwr_device.hpp"
#include "cwr_pack.hpp"

namespace cwr {

typedef unsigned long long u64;

constexpr int kLaneElems = 16;  // elements a lane holds of a chunk

// How a softmax at temperature T is evaluated: exponents in bits, t = x * c with c = log2(e) / T.
struct Temper {
    float c;     // log2(e) / T
    double inv;  // 1 / T
    double sq;   // T^2
};

template <typename T> struct RowPacks {
    static constexpr int VEC = Elem<T>::VEC;
    static constexpr int NP = kLaneElems / VEC;  // packs a lane holds
};

// elements in front of the first 16-byte boundary grid point at or before p
template <typename T> __device__ __forceinline__ int grid_offset(const T* p) {
    return (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
}

// The pack of row elements [e, e + VEC).  EDGE = false: rows are whole packs on the 16-byte grid; a pack outside
// the row comes back as -inf.  EDGE = true: a pack that sticks out of the row is read whole where it lies on the
// grid (its 16 bytes hold an element of the row, so they are memory of the same allocation; what is not
// the row's is struck out by mask_chunk or never used), and element by element where it does not.
template <typename T, bool EDGE, bool NT>
__device__ __forceinline__ v4i load_pack(const T* __restrict__ row, int e, int V) {
    constexpr int VEC = Elem<T>::VEC;
    v4i r = Pack<T>::neg_inf();
    if (!EDGE) {
        // an unsigned 32-bit byte offset (V < 2^28) next to the row's base: no 64-bit address per lane
        if (e < V) r = load_raw<NT>(reinterpret_cast<const char*>(row) + (unsigned)e * (unsigned)sizeof(T));
        return r;
    }
    // a row off the element grid of 16 bytes: the hardware takes any element-aligned address
    typedef v4i v4i_any __attribute__((aligned(2)));
    const bool some = e + VEC > 0 && e < V, whole = e >= 0 && e + VEC <= V;
    const bool grid = (reinterpret_cast<uintptr_t>(row + e) & 15) == 0;
    if (whole || (some && grid)) {
        r = *reinterpret_cast<const v4i_any*>(row + e);
    } else if (some) {
        PackT<T, VEC> p;
        __builtin_memcpy(&p, &r, 16);
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if ((unsigned)(e + j) < (unsigned)V) p.e[j] = row[e + j];
        __builtin_memcpy(&r, &p, 16);
    }
    return r;
}

// Elements of a chunk that lie outside the row become -inf (EDGE rows; the others' packs are whole).
template <typename T, int G, bool EDGE>
__device__ __forceinline__ void mask_chunk(float (&v)[kLaneElems], int e0, int l, int V) {
    constexpr int VEC = Elem<T>::VEC;
    if (!EDGE || (G == 64 && e0 >= 0 && e0 + 64 * kLaneElems <= V)) return;
#pragma unroll
    for (int s = 0; s < kLaneElems; ++s) {
        const int e = e0 + ((s / VEC) * G + l) * VEC + (s & (VEC - 1));
        v[s] = (unsigned)e < (unsigned)V ? v[s] : -INFINITY;
    }
}

// The packs of lane l of a group of G that make up the chunk whose first pack covers row elements [e0, ..).
template <typename T, int G, bool EDGE, bool NT>
__device__ __forceinline__ void load_chunk(const T* __restrict__ row, int e0, int l, int V, v4i (&raw)[RowPacks<T>::NP]) {
    constexpr int VEC = RowPacks<T>::VEC, NP = RowPacks<T>::NP;
    if (G == 64 && e0 >= 0 && e0 + 64 * kLaneElems <= V) {  // wholly inside the row: nothing to check
        typedef v4i v4i_any __attribute__((aligned(2)));
        const char* base = reinterpret_cast<const char*>(row) + (size_t)((unsigned)e0 * (unsigned)sizeof(T));
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const char* p = base + (unsigned)l * 16u + 1024u * i;
            if (EDGE) raw[i] = *reinterpret_cast<const v4i_any*>(p);
            else raw[i] = load_raw<NT>(p);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) raw[i] = load_pack<T, EDGE, NT>(row, e0 + (i * G + l) * VEC, V);
}

template <typename T>
__device__ __forceinline__ void unpack_chunk(const v4i (&raw)[RowPacks<T>::NP], float (&v)[kLaneElems]) {
    constexpr int VEC = RowPacks<T>::VEC;
#pragma unroll
    for (int i = 0; i < RowPacks<T>::NP; ++i) {
        float t[VEC];
        Pack<T>::unpack(raw[i], t);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i * VEC + j] = t[j];
    }
}

// ---------------------------------------------------------------------------------------------
// reductions over aligned groups of W lanes
// ---------------------------------------------------------------------------------------------
struct OpMaxI { static __device__ __forceinline__ int apply(int a, int b) { return a > b ? a : b; } };
struct OpMinI { static __device__ __forceinline__ int apply(int a, int b) { return a < b ? a : b; } };

// A whole wave reduced by the vector unit alone: operations whose first operand comes through DPP, six of
// them, the last lane then holds the result.  Written out because the compiler makes a move, a quieting
// maximum and the operation out of each.  A DPP operand has to be two wait states old.
#define CWR_WAVE_REDUCE(OP, v)                                                        \
    asm("s_nop 1\n\t" OP " %0, %0, %0 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n\t" \
        "s_nop 1\n\t" OP " %0, %0, %0 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n\t" \
        "s_nop 1\n\t" OP " %0, %0, %0 row_half_mirror row_mask:0xf bank_mask:0xf\n\t"     \
        "s_nop 1\n\t" OP " %0, %0, %0 row_mirror row_mask:0xf bank_mask:0xf\n\t"          \
        "s_nop 1\n\t" OP " %0, %0, %0 row_bcast:15 row_mask:0xa bank_mask:0xf\n\t"        \
        "s_nop 1\n\t" OP " %0, %0, %0 row_bcast:31 row_mask:0xc bank_mask:0xf\n\t"        \
        "s_nop 1"                                                                     \
        : "+v"(v))
__device__ __forceinline__ float wave_max(float v) {
    CWR_WAVE_REDUCE("v_max_f32_dpp", v);
    return readlane_f32(v, 63);
}
__device__ __forceinline__ float wave_min(float v) {
    CWR_WAVE_REDUCE("v_min_f32_dpp", v);
    return readlane_f32(v, 63);
}
__device__ __forceinline__ float wave_sum(float v) {
    CWR_WAVE_REDUCE("v_add_f32_dpp", v);
    return readlane_f32(v, 63);
}
template <int W> __device__ __forceinline__ float row_max(float v) {
    if constexpr (W == 64) return wave_max(v);
    else return group_allreduce<W, OpMax>(v);
}
template <int W> __device__ __forceinline__ float row_sum(float v) {
    if constexpr (W == 64) return wave_sum(v);
    else return group_allreduce<W, OpSum>(v);
}

template <int W, class Op>
__device__ __forceinline__ int group_allreduce_i32(int v) {
    if (W >= 2) v = Op::apply(v, dpp_i32<DPP_QUAD_XOR1>(v, v));
    if (W >= 4) v = Op::apply(v, dpp_i32<DPP_QUAD_XOR2>(v, v));
    if (W >= 8) v = Op::apply(v, dpp_i32<DPP_ROW_HALF_MIRROR>(v, v));
    if (W >= 16) v = Op::apply(v, dpp_i32<DPP_ROW_MIRROR>(v, v));
    if (W >= 32) v = Op::apply(v, __shfl_xor(v, 16));
    if (W >= 64) v = Op::apply(v, __shfl_xor(v, 32));
    return v;
}

template <int W> __device__ __forceinline__ double group_sum_f64(double v) {
#pragma unroll
    for (int d = 1; d < W; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

// Orders what the lanes of one wave write to LDS before what its other lanes read there.  A wave's LDS
// accesses are performed in order; this keeps the compiler from moving them.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// ---------------------------------------------------------------------------------------------
// running softmax statistics of a row, in bits
// ---------------------------------------------------------------------------------------------
// s = sum of 2^t and u = sum of 2^t t over the elements seen, t = x c - m c, m the largest x seen
// (-inf: none seen, or nothing but -inf; s and u are then 0).  m is the same in all lanes of the row.
struct Online {
    float m, s, u;
};

// What elements are measured against: t = fma(x - sub, c, -ms).  Normally sub = 0 and ms = m c rounded to fp32: one
// fma per element, and what the rounding loses is the same for the whole row and comes back exactly from an
// fma (ms_slip).  It also stands in every exponent, as a factor 2^slip of the row's sum, so it has to stay
// a small fraction of a bit: from |m c| = 2^16 on, where it could be more than 2^-9, m is subtracted first and the
// sum's largest term is 1.  (Rows and chunks masked with a finite constant, logits far from zero, small
// temperatures.)  A sum is then never below 1 - 2^-9, where the series of log2_of_sum is as exact as above 1.
struct Anchor {
    float sub, ms;
};
__device__ __forceinline__ bool far_off(float m, float c) { return !(fabsf(m * c) < 0x1p16f); }  // NaN, inf too
__device__ __forceinline__ Anchor anchor(float m, float c) {
    Anchor a = {0.f, m * c};
    if (far_off(m, c)) {
        a.sub = m;
        a.ms = 0.f;
    }
    if (m == -INFINITY) a.sub = 0.f;  // nothing but -inf: t = -inf
    return a;
}
__device__ __forceinline__ float measure(float x, const Anchor& a, float c) { return fmaf(x - a.sub, c, -a.ms); }
__device__ __forceinline__ float ms_slip(float m, float c) {  // m c - ms
    return far_off(m, c) ? 0.f : fmaf(m, c, -(m * c));
}
// How far, in bits, what is measured against `from` lies below what is measured against `to` >= from: the difference
// of ms where there is one, of m c where it was subtracted exactly.  Products as they are rounded in `anchor`:
// contracted into an fma the difference would be off by a slip.
__device__ __forceinline__ float anchor_shift(float from, float to, float c) {
#pragma clang fp contract(off)
    if (from == to) return 0.f;
    if (from == -INFINITY) return -INFINITY;  // nothing was there
    const bool far_from = far_off(from, c), far_to = far_off(to, c);
    const float mf = from * c, mt = to * c;
    if (!far_from && !far_to) return mf - mt;
    const double a = far_from ? (double)from * (double)c : (double)mf;
    const double b = far_to ? (double)to * (double)c : (double)mt;
    return (float)(a - b);
}

constexpr float kTFloor = -1024.f;  // 2^t is 0 far above it; keeps 0 * t finite where x is -inf

// the rare rows whose anchor has something to subtract first
template <int N> __device__ __forceinline__ void subtract_far(float (&v)[N], const Anchor& a) {
    if (__ballot(a.sub != 0.f) != 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] -= a.sub;
    }
}

template <bool ENTROPY, bool FAR>
__device__ __forceinline__ void online_chunk_as(const float (&v)[kLaneElems], const Anchor& a, float c, float& s, float& u) {
    float sa = 0.f, sb = 0.f, ua = 0.f, ub = 0.f;
#pragma unroll
    for (int i = 0; i < kLaneElems; i += 2) {
        const float t0 = FAR ? measure(v[i], a, c) : fmaf(v[i], c, -a.ms);
        const float t1 = FAR ? measure(v[i + 1], a, c) : fmaf(v[i + 1], c, -a.ms);
        const float e0 = fast_exp2(t0), e1 = fast_exp2(t1);
        sa += e0;
        sb += e1;
        if (ENTROPY) {
            ua = fmaf(e0, fmaxf(t0, kTFloor), ua);
            ub = fmaf(e1, fmaxf(t1, kTFloor), ub);
        }
    }
    s = sa + sb;
    u = ua + ub;
}
template <bool ENTROPY>
__device__ __forceinline__ void online_chunk(const float (&v)[kLaneElems], float m, float c, float& s, float& u) {
    const Anchor a = anchor(m, c);
    if (__ballot(a.sub != 0.f) != 0) online_chunk_as<ENTROPY, true>(v, a, c, s, u);
    else online_chunk_as<ENTROPY, false>(v, a, c, s, u);
}

// state o measured against a maximum mn at least as large
__device__ __forceinline__ void online_rebase(Online& o, float mn, float c) {
    if (o.m != mn) {
        const float d = fmaxf(anchor_shift(o.m, mn, c), kTFloor);
        const float f = fast_exp2(d);
        o.u = f * fmaf(o.s, d, o.u);
        o.s *= f;
        o.m = mn;
    }
}

// Largest of a lane's values, NaN left out where there is a number.  As three-way maxima written out: around
// fmaxf of values just loaded the compiler puts one more instruction per value, to quiet signalling NaNs.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ float chunk_max(const float (&v)[kLaneElems]) {
    const float a = max3(v[0], v[1], v[2]), b = max3(v[3], v[4], v[5]), c = max3(v[6], v[7], v[8]);
    const float d = max3(v[9], v[10], v[11]), e = max3(v[12], v[13], v[14]);
    return max3(max3(a, b, c), max3(d, e, v[15]), v[15]);
}

// log2 of the sum of 2^((x - m) c) from the sum s of 2^(x c - ms)
__device__ __forceinline__ float log2_sum(const Online& o, float c) { return log2_of_sum(o.s) - ms_slip(o.m, c); }

// ln p of the logit x in a row with maximum m and log2 sum l2.  The difference x - m is exact in 64 bits and
// the logarithm of the sum is small in a peaked row: the result keeps its absolute accuracy however
// large the logits are.  A row of nothing but -inf gives -inf.
__device__ __forceinline__ double logprob_f64(float x, float m, double l2, const Temper& tp) {
    if (x == -INFINITY && !(l2 != l2)) return -INFINITY;
    return ((double)x - (double)m) * tp.inv - l2 * 0.6931471805599453;
}
__device__ __forceinline__ float logprob(float x, float m, float l2, const Temper& tp) {
    return (float)logprob_f64(x, m, (double)l2, tp);
}

// log2 of a number >= 0: exact to about 1e-7, and next to 1 to as much of the result itself.  The exponent stands
// apart from the logarithm of the mantissa (as one fp32 number the logarithm of 1000 is off by 5e-7).
__device__ __forceinline__ double log2_f64(float s) {
    if (fabsf(s - 1.f) < 0.015625f) return (double)log2_of_sum(s);  // its series, on both sides of 1
    const float f = 2.f * __builtin_amdgcn_frexp_mantf(s);          // [1, 2)
    return (double)(__builtin_amdgcn_frexp_expf(s) - 1) + (double)log2_of_sum(f);
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
// Waves of 64 work-items a launch can hold: the runtime counts work-items in 32 bits.
constexpr i64 kMaxWaves = ((i64)1 << 26) - 64;

inline unsigned wave_blocks(i64 waves) {  // whole workgroups, a multiple of the XCDs
    return (unsigned)(((waves + kWavesPerBlock - 1) / kWavesPerBlock + 7) & ~(i64)7);
}

// rows of V elements, `stride` apart, are whole packs on the 16-byte grid
template <typename T> inline bool on_grid(const void* p, i64 stride, int V) {
    constexpr int VEC = Elem<T>::VEC;
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && V % VEC == 0 && stride % VEC == 0;
}

// Waves that share a row of `chunks` chunks: enough of them to fill 1024 SIMDs when there are few rows, as
// long as each has a chunk of its own.
inline int row_waves(i64 R, i64 chunks) { return chunks >= 16 && R < 1024 ? 16 : chunks >= 4 && R < 16384 ? 4 : 1; }

inline Temper make_temper(double temperature) {
    Temper tp;
    tp.c = (float)(1.4426950408889634 / temperature);
    tp.inv = 1.0 / temperature;
    tp.sq = temperature * temperature;
    return tp;
}

}  // namespace cwr
