// Scores straight from the joiner's rows: logits[r, v] = sum_k h[r, k] * W[v, k] + bias[v] are formed on
// the matrix cores a block of rows at a time, in fp32, and scored by the row kernels of scores.hip;
// the block is small enough to be read back from the caches it was written to, and the (R, V) logits never
// exist as a whole.
//
// Three shapes of the product, by its size:
//   few rows   (a decoding step) latency and reading the weight are what counts: a workgroup takes 32
//              vocabulary entries and 32 rows, its four waves a quarter of K each, operands go from memory
//              straight into the matrix instructions, and the four partial tiles meet in LDS;
//   hundreds   tiles of 64 x 64, both operands through LDS;
//   many rows  the walks of the fused output layer (cwr_joint_walk.hpp), resident rows for the
//              joint sizes that have them, streamed rows for any other multiple of 32, with the vocabulary
//              split over workgroups where the rows alone do not fill the GPU.
// The reference has no joiner.
#include "cwr_host.hpp"
#include "cwr_joint_walk.hpp"

namespace cwr {

// Finished blocks of a wave: its lanes hold 32 consecutive entries of a data row in either half (SWAP), so that
// a store writes two whole 128-byte lines (four entries of 32 rows per store instead, the other way round:
// 121 against 95 us for 62464 x 1024, H = 512).  Entries up to the row pitch are written; those beyond the
// vocabulary are -inf.
template <int NMV, int ND>
__device__ __forceinline__ void store_logits(const f32x16 (&acc)[NMV][ND], int v_first, int pitch, int hf, int l32, i64 row0,
                                             i64 R, float* __restrict__ out) {
#pragma unroll
    for (int nd = 0; nd < ND; ++nd) {
        float* base = out + (row0 + 32 * nd) * (i64)pitch;
        const bool all = row0 + 32 * nd + 32 <= R;
#pragma unroll
        for (int mv = 0; mv < NMV; ++mv) {
            const int v = v_first + 32 * mv + l32;
            if (v >= pitch) continue;
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (all || row0 + 32 * nd + acc_row(e, hf) < R)
                    base[acc_row(e, 0) * (i64)pitch + (4 * hf * pitch + v)] = acc[mv][nd][e];
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
    walk_resident<T, ND, KS, NMV, WAVES, RK, D2, true>(
        [&](v4i (&hreg)[ND][KS]) { load_resident_rows<T, ND, KS>(h, R, row0, hreg); }, W + (i64)v0 * (KS * 16),
        bias ? bias + v0 : nullptr, vn, lds, [&]() {},
        [&](const f32x16 (&acc)[NMV][ND], int v) { store_logits<NMV, ND>(acc, v0 + v, pitch, hf, l32, row0, R, out); });
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
    walk_streaming<T, TB, true>(h, W + (i64)v0 * H, bias ? bias + v0 : nullptr, R, H, vn, row0, lds,
                          [&](const f32x16 (&acc)[2][4], int v) {
                              store_logits<2, 4>(acc, v0 + v, pitch, hf, l32, row0 + 128 * wd, R, out);
                          });
}

// Few rows.  Operand fragments straight from memory: lane l32 of either half reads 16 bytes of weight row l32
// and of data row l32 per step of 16 along K; kAhead steps are in flight.  The four waves of a workgroup take a
// quarter of K each.
constexpr int kFewWaves = 4;

template <typename T, typename TB>
__global__ __launch_bounds__(64 * kFewWaves) void k_logits_few(const T* __restrict__ h, const T* __restrict__ W,
                                                               const TB* __restrict__ bias, i64 R, int H, int V, int pitch,
                                                               float* __restrict__ out) {
    constexpr int kAhead = 4;
    __shared__ __attribute__((aligned(16))) float part[kFewWaves][64 * 16];  // a 32x32 block over the lanes of a wave
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hf = lane >> 5, l32 = lane & 31;
    const int v0 = (int)blockIdx.x * 32;
    const i64 r = (i64)blockIdx.y * 32 + l32;
    // beyond the vocabulary or the rows: multiplied like the last one, dropped when stored
    const T* pw = W + (i64)(v0 + l32 < V ? v0 + l32 : V - 1) * H + 8 * hf;
    const T* ph = h + (r < R ? r : R - 1) * (i64)H + 8 * hf;
    const int steps = H / 16;
    const int s0 = steps * w / kFewWaves, s1 = steps * (w + 1) / kFewWaves;
    f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
    for (int s = s0; s < s1; s += kAhead) {
        v4i fa[kAhead], fb[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int at = 16 * (s + a < s1 ? s + a : s1 - 1);
            fa[a] = *reinterpret_cast<const v4i*>(pw + at);
            fb[a] = *reinterpret_cast<const v4i*>(ph + at);
        }
        __builtin_amdgcn_sched_barrier(0);  // all of a batch's loads go out before its first product waits
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const v4i none = {0, 0, 0, 0};
            acc = Mfma<T>::mac(s + a < s1 ? fa[a] : none, s + a < s1 ? fb[a] : none, acc);  // behind the last step: zeros
        }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
        *reinterpret_cast<float4*>(&part[w][(q * 64 + lane) * 4]) =
            make_float4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
    __syncthreads();
    // wave w finishes run w of every lane's four: the partial sums in a fixed order, then the bias
    const int v = v0 + acc_row(4 * w, hf);
    float4 sum = *reinterpret_cast<const float4*>(&part[0][(w * 64 + lane) * 4]);
#pragma unroll
    for (int k = 1; k < kFewWaves; ++k) {
        const float4 p = *reinterpret_cast<const float4*>(&part[k][(w * 64 + lane) * 4]);
        sum.x += p.x; sum.y += p.y; sum.z += p.z; sum.w += p.w;
    }
    float b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = v + e < V ? (bias ? Elem<TB>::to_f32(bias[v + e]) : 0.f) : -INFINITY;
    if (r < R && v < pitch)
        *reinterpret_cast<float4*>(out + r * (i64)pitch + v) =
            make_float4(sum.x + b[0], sum.y + b[1], sum.z + b[2], sum.w + b[3]);
}

// Hundreds of rows.  A workgroup of four waves takes 64 rows and 64 vocabulary entries, a quarter tile per wave;
// both operands pass through LDS in K-slabs of 64, read from memory as whole 128-byte lines two slabs ahead.
constexpr int kTileRows = 64, kTileV = 64, kSlab = 64, kSlabPitch = kSlab + 8;

template <typename T, typename TB>
__global__ __launch_bounds__(256) void k_logits_tile(const T* __restrict__ h, const T* __restrict__ W,
                                                     const TB* __restrict__ bias, i64 R, int H, int V, int pitch,
                                                     float* __restrict__ out) {
    __shared__ __attribute__((aligned(16))) T sh[2][kTileRows][kSlabPitch];
    __shared__ __attribute__((aligned(16))) T sw[2][kTileV][kSlabPitch];
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hf = lane >> 5, l32 = lane & 31;
    const int v0 = (int)blockIdx.x * kTileV;
    const i64 r0 = (i64)blockIdx.y * kTileRows;
    // thread t moves piece t % 8 (16 bytes) of rows t / 8 and t / 8 + 32 of either operand
    const int st_row = tid >> 3, st_k = (tid & 7) * 8;
    const T* src[4];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const i64 r = r0 + st_row + 32 * p;
        const int v = v0 + st_row + 32 * p;
        src[p] = h + (r < R ? r : R - 1) * (i64)H;       // rows and entries beyond the end are
        src[2 + p] = W + (i64)(v < V ? v : V - 1) * H;   // multiplied like the last one and dropped
    }
    struct Pre { v4i q[4]; };
    Pre pre[2];
    const int slabs = (H + kSlab - 1) / kSlab;
    auto fetch = [&](int s, Pre& p) {
        const int k = s * kSlab + st_k;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const v4i none = {0, 0, 0, 0};
            p.q[i] = k < H ? *reinterpret_cast<const v4i*>(src[i] + k) : none;  // half a slab at the end
        }
    };
    auto stage = [&](int b, const Pre& p) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            *reinterpret_cast<v4i*>(&sh[b][st_row + 32 * i][st_k]) = p.q[i];
            *reinterpret_cast<v4i*>(&sw[b][st_row + 32 * i][st_k]) = p.q[2 + i];
        }
    };
    const int wr = w & 1, wv = w >> 1;
    f32x16 acc[1][1];
    const int my_v = v0 + 32 * wv + l32;
    const float b = my_v < V ? (bias ? Elem<TB>::to_f32(bias[my_v]) : 0.f) : -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[0][0][e] = b;
    fetch(0, pre[0]);
    if (slabs > 1) fetch(1, pre[1]);
    stage(0, pre[0]);
    lds_barrier();
    auto slab = [&](int s, Pre& mine, Pre& next) {
        if (s + 2 < slabs) fetch(s + 2, mine);
#pragma unroll
        for (int ks = 0; ks < kSlab / 16; ++ks) {
            const v4i fa = *reinterpret_cast<const v4i*>(&sw[s & 1][32 * wv + l32][16 * ks + 8 * hf]);
            const v4i fb = *reinterpret_cast<const v4i*>(&sh[s & 1][32 * wr + l32][16 * ks + 8 * hf]);
            acc[0][0] = Mfma<T>::mac(fb, fa, acc[0][0]);
        }
        if (s + 1 < slabs) stage((s + 1) & 1, next);
        lds_barrier();
    };
    for (int s = 0; s < slabs; s += 2) {
        slab(s, pre[0], pre[1]);
        if (s + 1 < slabs) slab(s + 1, pre[1], pre[0]);
    }
    store_logits<1, 1>(acc, v0 + 32 * wv, pitch, hf, l32, r0 + 32 * wr, R, out);
}

// X(ND, H / 16, NMV, WAVES, RK, workgroups per CU, two register sets of weight loads in flight): the shapes of
// the fused output layer's forward pass, at H = 512 with two sets (loads issued behind a tile's stores return
// behind them, and a slice more of lead hides part of that: 62464 x 1024 took 95 -> 89 us on one box, 79 either way on
// another).  The flag here / the other way round, us, 62464 x 1024: H = 128 46 / 46, 192 48 / 70, 256 54 / 54, 320 62 / 88,
// 384 65 / 68, 448 74 / 102, 512 78 / 79, 576 93 / 126, 640 104 / 110, 704 135 / 262, 768 137 / 144, 832 150 / 425,
// 896 151 / 161, 960 170 / 498, 1024 166 / 175 (with an odd number of slices a tile the two sets take turns from tile
// to tile as well, and which is which is known at run time only).  H = 576 and 640 spill 6 and 28 registers and are still
// ahead of the streamed walk: 93 against 136 and 104 against 146 us (H = 128 46 / 65, 512 79 / 130, 1024 166 / 213).
#define CWR_LOGIT_SHAPES(X) X(1, 8, 4, 8, 64, 1, true) X(1, 12, 4, 8, 64, 1, false) X(1, 16, 4, 8, 64, 1, true) \
                            X(1, 20, 4, 8, 64, 1, false) X(1, 24, 4, 8, 64, 1, true) X(1, 28, 4, 8, 64, 1, false) \
                            X(1, 32, 4, 8, 64, 1, true) X(1, 36, 4, 8, 64, 1, false) X(1, 40, 4, 8, 64, 1, false) \
                            X(1, 44, 4, 4, 64, 1, false) X(1, 48, 4, 4, 64, 1, true) X(1, 52, 4, 4, 64, 1, false) \
                            X(1, 56, 4, 4, 64, 1, true) X(1, 60, 4, 4, 64, 1, false) X(1, 64, 4, 4, 64, 1, true)

// Vocabulary entries per workgroup, whole tiles of 128: as many parts as fit on the GPU at once (`resident`
// workgroups), since every part loads its rows anew and a second, partly filled round costs a whole one.
static int split_vocabulary(i64 row_blocks, i64 resident, int V, unsigned* splits) {
    const int tiles = (V + 127) / 128;
    i64 want = resident / row_blocks;
    want = want < 1 ? 1 : want > tiles ? tiles : want;
    const int per = (int)((tiles + want - 1) / want);
    *splits = (unsigned)((tiles + per - 1) / per);
    return per * 128;
}

template <typename T, typename TB>
static int logits_typed(const T* h, const T* w, const TB* bias, i64 R, int H, int V, int pitch, float* out,
                        hipStream_t stream) {
    // By the number of logits, which moves both borders little with the joint size (us, few / tiled / walked; bf16):
    //   V = 1024          R * V = 0.2e6       0.4e6            1.6e6             6e6                12e6
    //     H = 128       4.8 / 4.6 / 8.0   5.3 / 4.7 / 8.0   12 / 6.7 / 9.8   32 / 18.3 / 13.1   52 / 17 / 15
    //     H = 512       5.2 / 6.7 / 15    6.9 / 6.8 / 16    18 / 9.5 / 18    49 / 18.3 / 19.4   94 / 32 / 27
    //     H = 1024      6.7 / 9.1 / 18    10 / 9.6 / 18     29 / 15 / 19     90 / 30 / 30      175 / 52 / 49
    //   V = 4096, H = 640 5.9 / 7.2 / 16  8.6 / 7.2 / 17    24 / 10.5 / 22   71 / 21 / 25      137 / 37 / 37
    //   V = 300, H = 1056 5.8 / 9.7 / 31  9.1 / 10 / 32     36 / 17 / 37    125 / 42 / 41      240 / 80 / 50 (streamed)
    if (R * V <= 400000) {
        CWR_LAUNCH((k_logits_few<T, TB>), dim3((unsigned)((V + 31) / 32), (unsigned)((R + 31) / 32)), dim3(64 * kFewWaves),
                   0, stream, h, w, bias, R, H, V, pitch, out);
        return check_launch();
    }
    if (R * V <= 12000000 && R <= 64 * 65535) {
        CWR_LAUNCH((k_logits_tile<T, TB>), dim3((unsigned)((V + kTileV - 1) / kTileV),
                   (unsigned)((R + kTileRows - 1) / kTileRows)), dim3(256), 0, stream, h, w, bias, R, H, V, pitch, out);
        return check_launch();
    }
    unsigned splits;
#define CWR_LOGIT_RES(ND, KS, NMV, WAVES, RK, OCC, D2)                                                              \
    if (H == 16 * KS) {                                                                                             \
        const i64 blocks = (R + 32 * ND * WAVES - 1) / (32 * ND * WAVES);                                           \
        if (blocks > 0x7fffffffLL) return CWR_ERR_TOO_LARGE;                                                        \
        const int per = split_vocabulary(blocks, 256, V, &splits);                                                  \
        CWR_LAUNCH((k_logits_res<T, TB, ND, KS, NMV, WAVES, RK, OCC, D2>), dim3((unsigned)blocks, splits),          \
                   dim3(64 * WAVES), 0, stream, h, w, bias, R, V, pitch, per, out);                                 \
        return check_launch();                                                                                      \
    }
    CWR_LOGIT_SHAPES(CWR_LOGIT_RES)
#undef CWR_LOGIT_RES
    const i64 blocks = (R + kJM - 1) / kJM;
    if (blocks > 0x7fffffffLL) return CWR_ERR_TOO_LARGE;
    const int per = split_vocabulary(blocks, 512, V, &splits);
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

// Rows of logits that exist at a time: as many as the resident walk multiplies in one round of the GPU's 256
// CUs, unless that is more than a quarter of a GiB.
constexpr i64 kBlockRows = 65536, kBlockMinRows = 4096;
constexpr i64 kBlockBytes = (i64)256 << 20;

static i64 logit_pitch(i64 V) { return (V + 3) & ~(i64)3; }

size_t joint_scores_workspace_bytes(i64 R, i64 V) {
    const i64 row = logit_pitch(V) * 4;
    i64 rows = kBlockBytes / row;
    rows = rows < kBlockMinRows ? kBlockMinRows : rows > kBlockRows ? kBlockRows : rows;
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
