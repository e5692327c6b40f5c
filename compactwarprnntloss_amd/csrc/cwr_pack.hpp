// 16-byte accesses of the streaming kernels (raw packs and their fp32 values) and the numbering of
// their workgroups.
#pragma once

#include "cwr_device.hpp"

namespace cwr {

constexpr int kWavesPerBlock = 4;

typedef int v4i __attribute__((ext_vector_type(4)));

template <bool NT>
__device__ __forceinline__ v4i load_raw(const void* p) {
    const v4i* q = static_cast<const v4i*>(p);
    return NT ? __builtin_nontemporal_load(q) : *q;
}
template <bool NT>
__device__ __forceinline__ void store_raw(void* p, v4i v) {
    v4i* q = static_cast<v4i*>(p);
    if (NT) store_streaming_16(q, v); else *q = v;
}

// 16-byte pack <-> VEC fp32 values
template <typename T> struct Pack;
template <> struct Pack<float> {
    static __device__ __forceinline__ void unpack(v4i r, float (&o)[4]) {
        o[0] = __int_as_float(r.x); o[1] = __int_as_float(r.y); o[2] = __int_as_float(r.z); o[3] = __int_as_float(r.w);
    }
    static __device__ __forceinline__ v4i pack(const float (&i)[4]) {
        v4i r = {__float_as_int(i[0]), __float_as_int(i[1]), __float_as_int(i[2]), __float_as_int(i[3])};
        return r;
    }
    static __device__ __forceinline__ v4i neg_inf() {
        v4i r = {(int)0xff800000, (int)0xff800000, (int)0xff800000, (int)0xff800000};
        return r;
    }
};
template <> struct Pack<__half> {
    static __device__ __forceinline__ void unpack(v4i r, float (&o)[8]) {
        const int w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            __half2 h = *reinterpret_cast<const __half2*>(&w[j]);
            float2 f = __half22float2(h);
            o[2 * j] = f.x; o[2 * j + 1] = f.y;
        }
    }
    static __device__ __forceinline__ v4i pack(const float (&i)[8]) {
        int w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            __half2 h = __floats2half2_rn(i[2 * j], i[2 * j + 1]);
            w[j] = *reinterpret_cast<const int*>(&h);
        }
        v4i r = {w[0], w[1], w[2], w[3]};
        return r;
    }
    static __device__ __forceinline__ v4i neg_inf() {
        v4i r = {(int)0xfc00fc00, (int)0xfc00fc00, (int)0xfc00fc00, (int)0xfc00fc00};
        return r;
    }
};
template <> struct Pack<bf16_t> {
    static __device__ __forceinline__ void unpack(v4i r, float (&o)[8]) {
        const int w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o[2 * j] = __int_as_float(w[j] << 16);
            o[2 * j + 1] = __int_as_float(w[j] & (int)0xffff0000);
        }
    }
    static __device__ __forceinline__ v4i pack(const float (&i)[8]) {
        int w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            unsigned lo = Elem<bf16_t>::from_f32(i[2 * j]).v, hi = Elem<bf16_t>::from_f32(i[2 * j + 1]).v;
            w[j] = (int)(lo | (hi << 16));
        }
        v4i r = {w[0], w[1], w[2], w[3]};
        return r;
    }
    static __device__ __forceinline__ v4i neg_inf() {
        v4i r = {(int)0xff80ff80, (int)0xff80ff80, (int)0xff80ff80, (int)0xff80ff80};
        return r;
    }
};
template <> struct Pack<double> {
    static __device__ __forceinline__ void unpack(v4i r, float (&o)[2]) {
        o[0] = (float)__hiloint2double(r.y, r.x);
        o[1] = (float)__hiloint2double(r.w, r.z);
    }
    static __device__ __forceinline__ v4i pack(const float (&i)[2]) {
        double a = (double)i[0], b = (double)i[1];
        v4i r = {__double2loint(a), __double2hiint(a), __double2loint(b), __double2hiint(b)};
        return r;
    }
    static __device__ __forceinline__ v4i neg_inf() {
        v4i r = {0, (int)0xfff00000, 0, (int)0xfff00000};
        return r;
    }
};

// Workgroups are handed to the 8 XCDs round-robin.  With XCD_CONTIGUOUS the grid (a multiple of 8
// workgroups) is renumbered so that each XCD walks its own contiguous eighth of the rows: the
// small per-row outputs of neighbouring rows then meet in ONE L2 and leave it as full lines,
// instead of as eight partial lines from eight L2s.
template <bool XCD_CONTIGUOUS>
__device__ __forceinline__ i64 logical_block() {
    if (!XCD_CONTIGUOUS) return blockIdx.x;
    const unsigned per_xcd = gridDim.x >> 3;
    return (i64)(blockIdx.x & 7u) * per_xcd + (blockIdx.x >> 3);
}

// first row of this wave; wave-uniform by construction, and told so to the compiler so that the
// row decode of a one-row wave runs on the scalar unit
template <bool XCD_CONTIGUOUS = false>
__device__ __forceinline__ i64 wave_first_row(int rows_per_wave) {
    const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    return (logical_block<XCD_CONTIGUOUS>() * kWavesPerBlock + w) * rows_per_wave;
}

}  // namespace cwr
