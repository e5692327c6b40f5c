// Distillation of rows of logits from a teacher's top logits, forward and backward.
//
// Per row, z = x / T, p = softmax(z), and a list of K teacher entries (index i_k, value t_k):
//   without a tail  q = softmax(t / T) over the list,
//                   loss = T^2 sum_k q_k (log q_k - log p_{i_k})
//   with a tail     t_k = log q_k; what the list leaves, q_r = 1 - sum q, is one more class, and so is the
//                   student's mass outside the list, p_r = sum of p over entries not listed:
//                   loss = T^2 [ sum_k q_k (log q_k - log p_{i_k}) + q_r (log q_r - log p_r) ]
// The factor T^2 keeps the gradient's size when T changes.  With Q = sum q (+ q_r):
//   dx_v = g T [ p_v Q - sum_{k: i_k = v} q_k - (v not listed) q_r p_v / p_r ].
// For a transducer the list (blank, label) with a tail is the collapsed three-class distillation of
// a lattice cell.  The reference has no counterpart.
//
// Bound: HBM.  One read of the logits forward, one read and one write backward.
//
// p_r is summed over the entries outside the list, never formed as 1 - sum p: a confident student
// would leave nothing but rounding.  The listed entries are struck out of the registers that hold the
// row (a 16-bit mark per lane, set by the lane that holds the list entry), the rest is reduced with its own
// maximum, and the total is that plus the K listed logits.
#include "cwr_host.hpp"
#include "cwr_rowwalk.hpp"

namespace cwr {

struct DistillArgs {
    const float* top;  // (R, K)
    const int* index;  // (R, K), -1: absent
    int K;
    float* loss;   // (R)
    float4* stat;  // (R) what the backward pass needs; may be null
    int* status;   // may be null
};

// A lane's entry of the list: x its student logit, t the teacher's value
struct Entry {
    int at;  // -1: none
    float t, x;
    bool bad;
};

template <typename T>
__device__ __forceinline__ Entry load_entry(const T* __restrict__ row, i64 r, int l, int V, const float* __restrict__ top,
                                            const int* __restrict__ index, int K) {
    Entry e = {-1, -INFINITY, -INFINITY, false};
    if (l < K) {
        const int at = index[r * K + l];
        const float t = top[r * K + l];
        if ((unsigned)at < (unsigned)V) {
            e.at = at;
            e.t = t;
            e.x = Elem<T>::to_f32(row[at]);
        } else {
            e.bad = at != -1;
        }
    }
    return e;
}

// The teacher's probabilities of a row: q of this lane's entry, its logarithm, and the mass Q of the list.
template <int G, bool TAIL>
__device__ __forceinline__ void teacher(const Entry& e, const Temper& tp, float& q, float& logq, float& Q) {
    if (TAIL) {
        logq = e.t;
        q = fast_exp2(e.t * kLog2e);
        Q = row_sum<G>(q);
        return;
    }
    const float t = (float)((double)e.t * tp.inv);
    const float mt = row_max<G>(t);
    if (mt == -INFINITY) {  // an empty list, or one of -inf only
        q = t != t ? t : 0.f;
        logq = t;
        Q = row_sum<G>(q);
        return;
    }
    const float d = t - mt;
    const float ex = fast_exp2(d * kLog2e);
    const float s = row_sum<G>(ex);
    q = ex / s;
    logq = d - kLn2 * log2_of_sum(s);
    Q = s != s ? s : 1.f;
}

constexpr float kPoisoned = INFINITY;  // in place of a row's log2 sum: an index outside the vocabulary was met

// Everything behind the sums of a row, by the G lanes that share it.  o: the sums over the whole row, or with
// TAIL over the entries outside the list; first: this lane's entry is the one of its index that counts
template <int G, bool TAIL>
__device__ __forceinline__ void finish_row(i64 r, bool ok, int l, Online o, const Entry& e, bool first, const Temper& tp,
                                           const DistillArgs& a) {
    const float c = tp.c;
    float q, logq, Q;
    teacher<G, TAIL>(e, tp, q, logq, Q);
    const Online rest = o;
    if (TAIL) {
        online_rebase(o, fmaxf(o.m, row_max<G>(e.x)), c);
        o.s += row_sum<G>(first ? fast_exp2(measure(e.x, anchor(o.m, c), c)) : 0.f);
    }
    const bool empty = o.m == -INFINITY && !(o.s != o.s);
    const float l2 = empty ? 0.f : log2_sum(o, c);
    const float term = q == 0.f || e.at < 0 ? 0.f : q * (logq - logprob(e.x, o.m, l2, tp));
    float loss = row_sum<G>(term);
    float B = empty ? 0.f : Q * fast_exp2(-(l2 + ms_slip(o.m, c)));
    if (TAIL) {
        // the mass the list leaves in 64 bits: a list that holds nearly everything leaves a small difference
        const double left = 1.0 - group_sum_f64<G>(e.at >= 0 ? exp((double)e.t) : 0.0);
        const bool has_rest = rest.m > -INFINITY || rest.s != rest.s;
        const float qr = has_rest && left > 0.0 ? (float)left : 0.f;
        B = 0.f;
        if (has_rest) {
            const float l2r = log2_sum(rest, c);
            const float logpr = (float)(((double)rest.m - (double)o.m) * tp.inv +
                                        ((double)l2r - (double)l2) * 0.6931471805599453);
            if (qr > 0.f) loss += qr * (kLn2 * fast_log2(qr) - logpr);
            const float to_all = anchor_shift(rest.m, o.m, c) - (l2 + ms_slip(o.m, c));
            B = (Q + qr) * fast_exp2(to_all) - qr * fast_exp2(-(l2r + ms_slip(rest.m, c)));
        }
    }
    const bool bad = group_allreduce_i32<G, OpMaxI>(e.bad ? 1 : 0) != 0;
    if (bad && a.status) raise_flag(a.status, CWR_FLAG_BAD_LABEL);
    if (!ok || l != 0) return;
    a.loss[r] = bad ? __int_as_float(0x7fc00000) : loss / (float)(tp.inv * tp.inv);
    if (a.stat) a.stat[r] = bad ? make_float4(0.f, 0.f, 0.f, kPoisoned) : make_float4(rest.m, B, o.m, l2);
}

// G lanes per row (the row whole in registers), or one or NW waves per row that walk it in chunks.
template <typename T, int G, int NW, bool TAIL, bool EDGE>
__global__ __launch_bounds__(64 * (NW > 1 ? NW : kWavesPerBlock)) void k_distill(
    const T* __restrict__ x, i64 R, int V, i64 stride, const Temper tp, const DistillArgs a) {
    static_assert(NW == 1 || G == 64, "several waves share a row only as whole waves");
    constexpr int VEC = RowPacks<T>::VEC, NP = RowPacks<T>::NP, RP = 64 / G;
    constexpr int WB = NW > 1 ? NW : kWavesPerBlock;
    constexpr int CHUNK = G * kLaneElems;
    __shared__ unsigned marks[WB][64];
    __shared__ Online parts[WB];
    const int lane = threadIdx.x & 63, l = lane & (G - 1), g = lane / G;
    const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const i64 r0 = NW > 1 ? (i64)blockIdx.x : wave_first_row<true>(RP);
    if (r0 >= R) return;
    const i64 r = r0 + g;
    const bool ok = r < R;
    const i64 rr = ok ? r : R - 1;
    const T* row = x + rr * stride;
    const int off = EDGE ? grid_offset(row) : 0;
    const int first_chunk = NW > 1 ? w : 0;
    // G < 64: one chunk holds the row (the host sees to it)
    const int chunks = G < 64 ? 1 : (int)(((i64)V + off + CHUNK - 1) / CHUNK);

    v4i next[NP];
    auto fetch = [&](int ch) { load_chunk<T, G, EDGE, false>(row, ch * CHUNK - off, l, V, next); };
    if (first_chunk < chunks) fetch(first_chunk);
    const Entry e = load_entry<T>(row, rr, l, V, a.top, a.index, a.K);
    bool first = e.at >= 0;

    Online o = {-INFINITY, 0.f, 0.f};
    for (int ch = first_chunk; ch < chunks; ch += NW) {
        float v[kLaneElems];
        unpack_chunk<T>(next, v);
        mask_chunk<T, G, EDGE>(v, ch * CHUNK - off, l, V);
        if (G == 64 && ch + NW < chunks) fetch(ch + NW);
        if (TAIL) {
            marks[w][lane] = 0;
            wave_sync();
            const int place = e.at + off - ch * CHUNK;
            if (e.at >= 0 && place >= 0 && place < CHUNK) {
                const int pk = place / VEC;
                const unsigned bit = 1u << ((pk / G) * VEC + (place & (VEC - 1)));
                // of entries that name one index, the one that sets the mark counts
                first = (atomicOr(&marks[w][g * G + (pk & (G - 1))], bit) & bit) == 0;
            }
            wave_sync();
            const unsigned mine = marks[w][lane];
#pragma unroll
            for (int s = 0; s < kLaneElems; ++s) v[s] = (mine >> s) & 1 ? -INFINITY : v[s];
            wave_sync();
        }
        const float top = row_max<G>(chunk_max(v));
        if (G < 64) o.m = top;
        else online_rebase(o, fmaxf(o.m, top), tp.c);
        float s, u;
        online_chunk<false>(v, o.m, tp.c, s, u);
        o.s += s;
    }
    o.s = row_sum<G>(o.s);
    if (NW > 1) {
        if (lane == 0) parts[w] = o;
        __syncthreads();
        if (w != 0) return;
        float m = parts[0].m;
#pragma unroll
        for (int i = 1; i < NW; ++i) m = fmaxf(m, parts[i].m);
        online_rebase(o, m, tp.c);
#pragma unroll
        for (int i = 1; i < NW; ++i) {
            Online p = parts[i];
            online_rebase(p, m, tp.c);
            o.s += p.s;
        }
        if (TAIL) {  // the marks were set by several waves: the first of equal indices counts
            first = e.at >= 0;
            for (int j = 0; j < a.K; ++j)
                if (__builtin_amdgcn_readlane(e.at, j) == e.at && j < lane) first = false;
        }
    }
    finish_row<G, TAIL>(r, ok, l, o, e, first, tp, a);
}

// ---------------------------------------------------------------------------------------------
// sum and mean of the rows' losses, in a fixed order, in 64 bits
// ---------------------------------------------------------------------------------------------
constexpr int kSumBlocks = 1024;
constexpr int kSumThreads = 256;

__device__ __forceinline__ double block_sum(double v) {
    __shared__ double parts[kSumThreads / 64];
    v = group_sum_f64<64>(v);
    if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < kSumThreads / 64; ++i) s += parts[i];
    return s;
}

__global__ __launch_bounds__(kSumThreads) void k_sum_rows(const float* __restrict__ v, i64 n, double* __restrict__ part) {
    double s = 0.0;
    const i64 step = (i64)gridDim.x * kSumThreads;
    for (i64 i = (i64)blockIdx.x * kSumThreads + threadIdx.x; i < n; i += 4 * step) {  // four loads in flight
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = i + j * step < n ? v[i + j * step] : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) s += (double)f[j];
    }
    s = block_sum(s);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

template <typename S>
__global__ __launch_bounds__(kSumThreads) void k_sum_mean(const S* __restrict__ v, i64 n, i64 R, float* __restrict__ sum,
                                                          float* __restrict__ mean) {
    double s = 0.0;
    for (i64 i = threadIdx.x; i < n; i += kSumThreads) s += (double)v[i];
    s = block_sum(s);
    if (threadIdx.x == 0) {
        if (sum) *sum = (float)s;
        if (mean) *mean = (float)(s / (double)R);
    }
}

size_t sum_workspace_bytes() { return kSumBlocks * sizeof(double); }

static int launch_sum_mean(const float* rows, i64 R, double* work, float* sum, float* mean, hipStream_t stream) {
    if (R <= 16 * kSumThreads) {
        CWR_LAUNCH((k_sum_mean<float>), dim3(1), dim3(kSumThreads), 0, stream, rows, R, R, sum, mean);
        return check_launch();
    }
    const i64 want = (R + 4 * kSumThreads - 1) / (4 * kSumThreads);
    const int blocks = want < kSumBlocks ? (int)want : kSumBlocks;
    CWR_LAUNCH(k_sum_rows, dim3((unsigned)blocks), dim3(kSumThreads), 0, stream, rows, R, work);
    const int rc = check_launch();
    if (rc != CWR_OK) return rc;
    CWR_LAUNCH((k_sum_mean<double>), dim3(1), dim3(kSumThreads), 0, stream, work, (i64)blocks, R, sum, mean);
    return check_launch();
}

// ---------------------------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------------------------
constexpr int kUnset = 0x7fedcba9;  // a NaN no arithmetic here produces: not an entry of the list

// One wave per chunk of a row (G = 64) or per 64 / G whole rows.  Outside the list the gradient is one
// exponential times a number of the row; each listed entry is worked out by one lane and put into a map
// of the chunk in LDS, from where the pass over the chunk picks it up, so that every element is written once.
template <typename T, int G, bool TAIL, bool EDGE>
__global__ __launch_bounds__(kWavesPerBlock * 64) void k_distill_grad(
    const T* __restrict__ x, i64 R, int V, i64 stride, const Temper tp, const float* __restrict__ top,
    const int* __restrict__ index, int K, const float4* __restrict__ stat, const GradOut go, int chunks_per_row,
    T* __restrict__ dx) {
    constexpr int VEC = RowPacks<T>::VEC, NP = RowPacks<T>::NP, RP = 64 / G;
    constexpr int CHUNK = G * kLaneElems;
    __shared__ __attribute__((aligned(16))) int map_[kWavesPerBlock][64 * kLaneElems];
    const int lane = threadIdx.x & 63, l = lane & (G - 1), g = lane / G;
    const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const i64 wave = wave_first_row<true>(1);
    i64 r;
    int ch = 0;
    if (G == 64) {
        if (wave >= R * chunks_per_row) return;
        r = chunks_per_row == 1 ? wave : wave / chunks_per_row;
        ch = (int)(wave - r * chunks_per_row);
    } else {
        r = wave * RP + g;
        if (wave * RP >= R) return;
    }
    const bool ok = r < R;
    if (!ok) r = R - 1;
    const T* row = x + r * stride;
    T* out = dx + r * (i64)V;
    const int off = EDGE ? grid_offset(out) : 0;  // the stores decide: a load may start anywhere
    const int e0 = ch * CHUNK - off;              // row element of map place 0
    v4i raw[NP];
    load_chunk<T, G, EDGE, false>(row, e0, l, V, raw);
    const Entry e = load_entry<T>(row, r, l, V, top, index, K);
    const float4 st = stat[r];
    float gt = go.p[r * go.stride] * go.scale / (float)tp.inv;
    int* map = map_[w] + g * CHUNK;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        int* p = map + (i * G + l) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) p[j] = kUnset;
    }
    float q, logq, Q;
    teacher<G, TAIL>(e, tp, q, logq, Q);
    if (TAIL && (st.x > -INFINITY)) Q = fmaxf(Q, 1.f);  // with the tail's mass, where there is a tail
    const float c = tp.c;
    const Anchor ref = anchor(st.x, c);
    const bool poisoned = st.w == kPoisoned;
    const float B = poisoned ? 0.f : st.y * gt;
    wave_sync();
    const int place = e.at - e0;
    const bool here = e.at >= 0 && place >= 0 && place < CHUNK;
    if (here) map[place] = lane;
    wave_sync();
    if (__ballot(here && map[place] != lane) != 0) {  // an index listed more than once: its shares add up, in order
        float sum = 0.f;
        for (int j = 0; j < K; ++j) {
            const float qj = __shfl(q, g * G + j);
            const int aj = __shfl(e.at, g * G + j);
            sum += aj == e.at ? qj : 0.f;
        }
        q = sum;
    }
    wave_sync();
    if (here) {
        const bool empty = st.z == -INFINITY && st.w == st.w;
        const float p = empty ? 0.f : fast_exp2(measure(e.x, anchor(st.z, c), c) - (st.w + ms_slip(st.z, c)));
        map[place] = poisoned ? 0 : __float_as_int(gt * fmaf(p, Q, -q));
    }
    wave_sync();
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int p0 = (i * G + l) * VEC, el = e0 + p0;
        float v[VEC], d[VEC];
        Pack<T>::unpack(raw[i], v);
        subtract_far(v, ref);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float dense = fast_exp2(fmaf(v[j], c, -ref.ms)) * B;
            const int given = map[p0 + j];
            d[j] = given != kUnset ? __int_as_float(given) : dense;
        }
        if (poisoned) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) d[j] = 0.f;
        }
        if (!ok || el >= V) continue;
        if (!EDGE || (el >= 0 && el + VEC <= V)) {
            store_raw<G == 64 || (!EDGE && G >= 8)>(out + el, Pack<T>::pack(d));
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if ((unsigned)(el + j) < (unsigned)V) out[el + j] = Elem<T>::from_f32(d[j]);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------
template <typename T, bool TAIL, bool EDGE>
static int distill_typed(const T* x, i64 R, int V, i64 stride, const Temper& tp, const DistillArgs& a,
                         hipStream_t stream) {
    const int span = V + (EDGE ? RowPacks<T>::VEC - 1 : 0);  // places a row can take on the pack grid
    int G = 4;
    while (G < 64 && (G * kLaneElems < span || G < a.K)) G *= 2;  // a lane for every list entry
#define CWR_GROUP(GG)                                                                                               \
    if (G == GG) {                                                                                                  \
        const i64 waves = (R + 64 / GG - 1) / (64 / GG);                                                            \
        if (waves > 0x3fffffffLL * kWavesPerBlock) return CWR_ERR_TOO_LARGE;                                        \
        CWR_LAUNCH((k_distill<T, GG, 1, TAIL, EDGE>), dim3(wave_blocks(waves)), dim3(kWavesPerBlock * 64), 0, stream, \
                   x, R, V, stride, tp, a);                                                                         \
        return check_launch();                                                                                      \
    }
    CWR_GROUP(4) CWR_GROUP(8) CWR_GROUP(16) CWR_GROUP(32)
    const i64 chunks = ((i64)span + 64 * kLaneElems - 1) / (64 * kLaneElems);
    const int NW = row_waves(R, chunks);
    if (R > 0x3fffffffLL) return CWR_ERR_TOO_LARGE;
    if (NW == 1) { CWR_GROUP(64) }
#undef CWR_GROUP
    if (NW == 16)
        CWR_LAUNCH((k_distill<T, 64, 16, TAIL, EDGE>), dim3((unsigned)R), dim3(1024), 0, stream, x, R, V, stride, tp, a);
    else
        CWR_LAUNCH((k_distill<T, 64, 4, TAIL, EDGE>), dim3((unsigned)R), dim3(256), 0, stream, x, R, V, stride, tp, a);
    return check_launch();
}

template <typename T, bool TAIL, bool EDGE>
static int distill_grad_typed(const T* x, i64 R, int V, i64 stride, const Temper& tp, const RowDistill& s, const GradOut& go,
                              T* dx, hipStream_t stream) {
    const int span = V + (EDGE ? RowPacks<T>::VEC - 1 : 0);
    int G = 4;
    while (G < 64 && (G * kLaneElems < span || G < s.K)) G *= 2;
    const i64 chunks = G < 64 ? 1 : ((i64)span + 64 * kLaneElems - 1) / (64 * kLaneElems);
    const i64 waves = G < 64 ? (R + 64 / G - 1) / (64 / G) : R * chunks;
    if (waves > 0x3fffffffLL * kWavesPerBlock) return CWR_ERR_TOO_LARGE;
#define CWR_GROUP(GG)                                                                                                  \
    if (G == GG)                                                                                                       \
        CWR_LAUNCH((k_distill_grad<T, GG, TAIL, EDGE>), dim3(wave_blocks(waves)), dim3(kWavesPerBlock * 64), 0, stream, \
                   x, R, V, stride, tp, s.top, s.index, (int)s.K, reinterpret_cast<const float4*>(s.stat), go,          \
                   (int)chunks, dx);
    CWR_GROUP(4) CWR_GROUP(8) CWR_GROUP(16) CWR_GROUP(32) CWR_GROUP(64)
#undef CWR_GROUP
    return check_launch();
}

template <typename T>
static int distill_any(const void* x, i64 R, int V, i64 stride, const Temper& tp, bool tail, const DistillArgs& a,
                       hipStream_t stream) {
    const T* p = static_cast<const T*>(x);
    const bool grid = on_grid<T>(x, stride, V);
    if (tail)
        return grid ? distill_typed<T, true, false>(p, R, V, stride, tp, a, stream)
                    : distill_typed<T, true, true>(p, R, V, stride, tp, a, stream);
    return grid ? distill_typed<T, false, false>(p, R, V, stride, tp, a, stream)
                : distill_typed<T, false, true>(p, R, V, stride, tp, a, stream);
}

template <typename T>
static int distill_grad_any(const void* x, i64 R, int V, i64 stride, const Temper& tp, const RowDistill& s,
                            const GradOut& go, void* dx, hipStream_t stream) {
    const T* p = static_cast<const T*>(x);
    T* d = static_cast<T*>(dx);
    const bool grid = on_grid<T>(x, stride, V) && on_grid<T>(dx, V, V);
    if (s.tail)
        return grid ? distill_grad_typed<T, true, false>(p, R, V, stride, tp, s, go, d, stream)
                    : distill_grad_typed<T, true, true>(p, R, V, stride, tp, s, go, d, stream);
    return grid ? distill_grad_typed<T, false, false>(p, R, V, stride, tp, s, go, d, stream)
                : distill_grad_typed<T, false, true>(p, R, V, stride, tp, s, go, d, stream);
}

int launch_distill(const void* x, int dtype, i64 R, i64 V, i64 stride, double temperature, const RowDistill& s,
                   float* loss, float* loss_sum, float* loss_mean, void* workspace, int* status, hipStream_t stream) {
    DistillArgs a;
    a.top = s.top; a.index = s.index; a.K = (int)s.K; a.loss = loss; a.stat = reinterpret_cast<float4*>(s.stat);
    a.status = status;
    const Temper tp = make_temper(temperature);
    int rc = CWR_OK;
    if (R > 0) {
        switch (dtype) {
            case CWR_F32: rc = distill_any<float>(x, R, (int)V, stride, tp, s.tail, a, stream); break;
            case CWR_F16: rc = distill_any<__half>(x, R, (int)V, stride, tp, s.tail, a, stream); break;
            case CWR_BF16: rc = distill_any<bf16_t>(x, R, (int)V, stride, tp, s.tail, a, stream); break;
            case CWR_F64: rc = distill_any<double>(x, R, (int)V, stride, tp, s.tail, a, stream); break;
            default: return CWR_ERR_DTYPE;
        }
    }
    if (rc != CWR_OK || (!loss_sum && !loss_mean)) return rc;
    return launch_sum_mean(loss, R, static_cast<double*>(workspace), loss_sum, loss_mean, stream);
}

int launch_distill_grad(const void* x, int dtype, i64 R, i64 V, i64 stride, double temperature, const RowDistill& s,
                        const GradOut go, void* dx, hipStream_t stream) {
    if (R == 0) return CWR_OK;
    const Temper tp = make_temper(temperature);
    switch (dtype) {
        case CWR_F32: return distill_grad_any<float>(x, R, (int)V, stride, tp, s, go, dx, stream);
        case CWR_F16: return distill_grad_any<__half>(x, R, (int)V, stride, tp, s, go, dx, stream);
        case CWR_BF16: return distill_grad_any<bf16_t>(x, R, (int)V, stride, tp, s, go, dx, stream);
        case CWR_F64: return distill_grad_any<double>(x, R, (int)V, stride, tp, s, go, dx, stream);
    }
    return CWR_ERR_DTYPE;
}

}  // namespace cwr
