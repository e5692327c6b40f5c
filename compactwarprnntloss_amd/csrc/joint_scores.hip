// Scores straight from the joiner's rows: logits[r, v] = sum_k h[r, k] * W[v, k] + bias[v] are formed on
// the matrix cores a block of rows at a time, in fp32, and scored by the row kernels of scores.hip;
// the block is small enough to be read back from the caches it was written to, and the (R, V) logits never
// exist as a whole.
//
// Three shapes of the product, by the number of rows:
//   few rows   (a decoding step) the weight is what has to be read: a workgroup takes 32 NVT vocabulary
//              entries and 32 NRT rows, its four waves a quarter of K each, operands go from memory
//              straight into the matrix instructions, and the four partial tiles meet in LDS;
//   many rows  the walks of the fused output layer (cwr_joint_walk.hpp), resident rows for the
//              joint sizes that have them, streamed rows for any other multiple of 32, with the vocabulary
//              split over workgroups where the rows alone do not fill the GPU.
// The reference has no joiner.
#include "cwr_host.hpp"
#include "cwr_joint_walk.hpp"

namespace cwr {

// Row r of a finished 32x32 block: the lane holds four runs of four entries of one data row.  Entries up to
// the row pitch are written (those beyond the vocabulary are -inf), so that every store is 16 bytes.
template <int NMV, int ND>
__device__ __forceinline__ void store_logits(const f32x16 (&acc)[NMV][ND], int v_first, int pitch, int hf, i64 rbase, i64 R,
                                             float* __restrict__ out) {
#pragma unroll
    for (int nd = 0; nd < ND; ++nd) {
        const i64 r = rbase + 32 * nd;
        if (r >= R) continue;
        float* row = out + r * (i64)pitch;
#pragma unroll
        for (int mv = 0; mv < NMV; ++mv)
#pragma unroll
            for (int b4 = 0; b4 < 4; ++b4) {
                const int v = v_first + 32 * mv + acc_row(4 * b4, hf);
                if (v < pitch)
                    *reinterpret_cast<float4*>(row + v) = make_float4(acc[mv][nd][4 * b4], acc[mv][nd][4 * b4 + 1],
                                                                      acc[mv][nd][4 * b4 + 2], acc[mv][nd][4 * b4 + 3]);
            }
    }
}

template <typename T, typename TB, int ND, int KS, int NMV, int WAVES, int RK, int OCC, bool D2>
__global__ __launch_bounds__(64 * WAVES, OCC) void k_logits_res(const T* __restrict__ h, const T* __restrict__ W,
                                                                const TB* __restrict__ bias, i64 R, int V, int pitch,
                                                                int v_per_split, float* __restrict__ out) {
    __shared__ __attribute__((aligned(16))) ResLds<T, NMV, RK> lds;
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hf = lane >> 5, l32 = lane & 31;
    const i64 row0 = (i64)blockIdx.x * (32 * ND * WAVES) + (i64)w * (32 * ND);
    const int v0 = (int)blockIdx.y * v_per_split;
    const int vn = V - v0 < v_per_split ? V - v0 : v_per_split;
    walk_resident<T, ND, KS, NMV, WAVES, RK, D2>(
        [&](v4i (&hreg)[ND][KS]) { load_resident_rows<T, ND, KS>(h, R, row0, hreg); }, W + (i64)v0 * (KS * 16),
        bias ? bias + v0 : nullptr, vn, lds, [&]() {},
        [&](const f32x16 (&acc)[NMV][ND], int v) { store_logits<NMV, ND>(acc, v0 + v, pitch, hf, row0 + l32, R, out); });
}

template <typename T, typename TB>
__global__ __launch_bounds__(256, 2) void k_logits_stream(const T* __restrict__ h, const T* __restrict__ W,
                                                          const TB* __restrict__ bias, i64 R, int H, int V, int pitch,
                                                          int v_per_split, float* __restrict__ out) {
    __shared__ __attribute__((aligned(16))) StreamLds<T> lds;
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wd = w & 1;
    const int hf = lane >> 5, l32 = lane & 31;
    const i64 row0 = (i64)blockIdx.x * kJM;
    const int v0 = (int)blockIdx.y * v_per_split;
    const int vn = V - v0 < v_per_split ? V - v0 : v_per_split;
    walk_streaming<T, TB>(h, W + (i64)v0 * H, bias ? bias + v0 : nullptr, R, H, vn, row0, lds,
                          [&](const f32x16 (&acc)[2][4], int v) {
                              store_logits<2, 4>(acc, v0 + v, pitch, hf, row0 + 128 * wd + l32, R, out);
                          });
}

// Few rows.  Operand fragments straight from memory: lane l32 of either half reads 16 bytes of weight row l32
// and of data row l32 per step of 16 along K; kAhead steps are in flight.
constexpr int kFewWaves = 4;

template <typename T, typename TB, int NRT, int NVT>
__global__ __launch_bounds__(64 * kFewWaves) void k_logits_few(const T* __restrict__ h, const T* __restrict__ W,
                                                               const TB* __restrict__ bias, i64 R, int H, int V, int pitch,
                                                               float* __restrict__ out) {
    constexpr int kAhead = 4;
    constexpr int TILE = 64 * 16;  // floats of a 32x32 block over the lanes of a wave
    __shared__ __attribute__((aligned(16))) float part[kFewWaves][NVT][NRT][TILE];
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hf = lane >> 5, l32 = lane & 31;
    const int v0 = (int)blockIdx.x * (32 * NVT);
    const i64 r0 = (i64)blockIdx.y * (32 * NRT);
    const T* pw[NVT];
    const T* ph[NRT];
#pragma unroll
    for (int i = 0; i < NVT; ++i) {
        const int v = v0 + 32 * i + l32;
        pw[i] = W + (i64)(v < V ? v : V - 1) * H + 8 * hf;  // beyond the vocabulary: dropped when stored
    }
#pragma unroll
    for (int j = 0; j < NRT; ++j) {
        const i64 r = r0 + 32 * j + l32;
        ph[j] = h + (r < R ? r : R - 1) * (i64)H + 8 * hf;
    }
    const int steps = H / 16;
    const int s0 = steps * w / kFewWaves, s1 = steps * (w + 1) / kFewWaves;
    f32x16 acc[NVT][NRT];
#pragma unroll
    for (int i = 0; i < NVT; ++i)
#pragma unroll
        for (int j = 0; j < NRT; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    for (int s = s0; s < s1; s += kAhead) {
        v4i fa[kAhead][NVT], fb[kAhead][NRT];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int at = 16 * (s + a < s1 ? s + a : s1 - 1);
#pragma unroll
            for (int i = 0; i < NVT; ++i) fa[a][i] = *reinterpret_cast<const v4i*>(pw[i] + at);
#pragma unroll
            for (int j = 0; j < NRT; ++j) fb[a][j] = *reinterpret_cast<const v4i*>(ph[j] + at);
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            if (s + a >= s1) break;
#pragma unroll
            for (int i = 0; i < NVT; ++i)
#pragma unroll
                for (int j = 0; j < NRT; ++j) acc[i][j] = Mfma<T>::mac(fa[a][i], fb[a][j], acc[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < NVT; ++i)
#pragma unroll
        for (int j = 0; j < NRT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<float4*>(&part[w][i][j][(q * 64 + lane) * 4]) =
                    make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
    __syncthreads();
    // wave w finishes run w of every lane's four: the partial sums in a fixed order, then the bias
#pragma unroll
    for (int i = 0; i < NVT; ++i) {
        const int v = v0 + 32 * i + acc_row(4 * w, hf);
        float b[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = v + e < V ? (bias ? Elem<TB>::to_f32(bias[v + e]) : 0.f) : -INFINITY;
#pragma unroll
        for (int j = 0; j < NRT; ++j) {
            const i64 r = r0 + 32 * j + l32;
            float4 sum = *reinterpret_cast<const float4*>(&part[0][i][j][(w * 64 + lane) * 4]);
#pragma unroll
            for (int k = 1; k < kFewWaves; ++k) {
                const float4 p = *reinterpret_cast<const float4*>(&part[k][i][j][(w * 64 + lane) * 4]);
                sum.x += p.x; sum.y += p.y; sum.z += p.z; sum.w += p.w;
            }
            if (r < R && v < pitch)
                *reinterpret_cast<float4*>(out + r * (i64)pitch + v) =
                    make_float4(sum.x + b[0], sum.y + b[1], sum.z + b[2], sum.w + b[3]);
        }
    }
}

// X(ND, H / 16, NMV, WAVES, RK, workgroups per CU, two register sets of weight loads in flight): the shapes of
// the fused output layer's forward pass
#define CWR_LOGIT_SHAPES(X) X(1, 8, 4, 8, 64, 1, true) X(1, 12, 4, 8, 64, 1, false) X(1, 16, 4, 8, 64, 1, true) \
                            X(1, 20, 4, 8, 64, 1, false) X(1, 24, 4, 8, 64, 1, true) X(1, 28, 4, 8, 64, 1, false) \
                            X(1, 32, 4, 8, 64, 1, false) X(1, 36, 4, 8, 64, 1, false) X(1, 40, 4, 8, 64, 1, false) \
                            X(1, 44, 4, 4, 64, 1, false) X(1, 48, 4, 4, 64, 1, true) X(1, 52, 4, 4, 64, 1, false) \
                            X(1, 56, 4, 4, 64, 1, true) X(1, 60, 4, 4, 64, 1, false) X(1, 64, 4, 4, 64, 1, true)

// vocabulary entries per workgroup, whole tiles of 128, so that `row_blocks` of them fill the GPU twice
static int split_vocabulary(i64 row_blocks, int V, unsigned* splits) {
    const int tiles = (V + 127) / 128;
    i64 want = (512 + row_blocks - 1) / row_blocks;
    want = want < 1 ? 1 : want > tiles ? tiles : want;
    const int per = (int)((tiles + want - 1) / want);
    *splits = (unsigned)((tiles + per - 1) / per);
    return per * 128;
}

template <typename T, typename TB>
static int logits_typed(const T* h, const T* w, const TB* bias, i64 R, int H, int V, int pitch, float* out,
                        hipStream_t stream) {
    if (R <= 1024) {
        if (R <= 32)
            CWR_LAUNCH((k_logits_few<T, TB, 1, 1>), dim3((unsigned)((V + 31) / 32), (unsigned)((R + 31) / 32)),
                       dim3(64 * kFewWaves), 0, stream, h, w, bias, R, H, V, pitch, out);
        else
            CWR_LAUNCH((k_logits_few<T, TB, 2, 2>), dim3((unsigned)((V + 63) / 64), (unsigned)((R + 63) / 64)),
                       dim3(64 * kFewWaves), 0, stream, h, w, bias, R, H, V, pitch, out);
        return check_launch();
    }
    unsigned splits;
#define CWR_LOGIT_RES(ND, KS, NMV, WAVES, RK, OCC, D2)                                                              \
    if (H == 16 * KS) {                                                                                             \
        const i64 blocks = (R + 32 * ND * WAVES - 1) / (32 * ND * WAVES);                                           \
        if (blocks > 0x7fffffffLL) return CWR_ERR_TOO_LARGE;                                                        \
        const int per = split_vocabulary(blocks, V, &splits);                                                       \
        CWR_LAUNCH((k_logits_res<T, TB, ND, KS, NMV, WAVES, RK, OCC, D2>), dim3((unsigned)blocks, splits),          \
                   dim3(64 * WAVES), 0, stream, h, w, bias, R, V, pitch, per, out);                                 \
        return check_launch();                                                                                      \
    }
    CWR_LOGIT_SHAPES(CWR_LOGIT_RES)
#undef CWR_LOGIT_RES
    const i64 blocks = (R + kJM - 1) / kJM;
    if (blocks > 0x7fffffffLL) return CWR_ERR_TOO_LARGE;
    const int per = split_vocabulary(blocks, V, &splits);
    CWR_LAUNCH((k_logits_stream<T, TB>), dim3((unsigned)blocks, splits), dim3(256), 0, stream, h, w, bias, R, H, V, pitch,
               per, out);
    return check_launch();
}

template <typename T>
static int logits_any(const void* h, const void* w, const void* bias, int bias_dtype, i64 R, int H, int V, int pitch,
                      float* out, hipStream_t stream) {
    const T* hp = static_cast<const T*>(h);
    const T* wp = static_cast<const T*>(w);
    if (bias_dtype == CWR_F32)
        return logits_typed<T, float>(hp, wp, static_cast<const float*>(bias), R, H, V, pitch, out, stream);
    return logits_typed<T, T>(hp, wp, static_cast<const T*>(bias), R, H, V, pitch, out, stream);
}

// Rows of logits that exist at a time.
constexpr i64 kBlockBytes = (i64)128 << 20;
constexpr i64 kBlockMinRows = 4096;

static i64 logit_pitch(i64 V) { return (V + 3) & ~(i64)3; }

size_t joint_scores_workspace_bytes(i64 R, i64 V) {
    const i64 row = logit_pitch(V) * 4;
    i64 rows = kBlockBytes / row;
    rows = rows < kBlockMinRows ? kBlockMinRows : rows;
    return (size_t)((R < rows ? R : rows) * row);
}

int launch_joint_scores(const void* h, const void* w, const void* bias, int bias_dtype, int dtype, i64 R, i64 H, i64 V,
                        double temperature, const RowScores& s, void* workspace, size_t workspace_bytes,
                        hipStream_t stream) {
    if (R == 0) return CWR_OK;
    const i64 pitch = logit_pitch(V);
    const i64 fit = (i64)(workspace_bytes / (size_t)(pitch * 4));
    if (fit < 1) return CWR_ERR_SHAPE;
    // equal blocks, whole workgroups of rows
    const i64 blocks = (R + fit - 1) / fit;
    i64 rows = (R + blocks - 1) / blocks;
    if (blocks > 1 && ((rows + 255) & ~(i64)255) <= fit) rows = (rows + 255) & ~(i64)255;
    float* logits = static_cast<float*>(workspace);
    const size_t es = 2;
    for (i64 r0 = 0; r0 < R; r0 += rows) {
        const i64 n = R - r0 < rows ? R - r0 : rows;
        const char* hp = static_cast<const char*>(h) + (size_t)(r0 * H) * es;
        int rc = dtype == CWR_BF16
                     ? logits_any<bf16_t>(hp, w, bias, bias_dtype, n, (int)H, (int)V, (int)pitch, logits, stream)
                     : logits_any<__half>(hp, w, bias, bias_dtype, n, (int)H, (int)V, (int)pitch, logits, stream);
        if (rc != CWR_OK) return rc;
        RowScores part = s;
        if (s.tokens) part.tokens = s.tokens + r0 * s.M;
        if (s.logprobs) part.logprobs = s.logprobs + r0 * s.M;
        if (s.entropy) part.entropy = s.entropy + r0;
        if (s.lse) part.lse = s.lse + r0;
        if (s.top_logprobs) part.top_logprobs = s.top_logprobs + r0 * s.K;
        if (s.top_index) part.top_index = s.top_index + r0 * s.K;
        rc = launch_scores(logits, CWR_F32, n, V, pitch, temperature, part, stream);
        if (rc != CWR_OK) return rc;
    }
    return CWR_OK;
}

}  // namespace cwr
