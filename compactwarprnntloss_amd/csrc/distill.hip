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

// An entry of the list: x its student logit, t the teacher's value.  Lane l of a group of G holds entries
// l, l + G, ..: E of them, so that a long list does not widen the group a short row needs.
struct Entry {
    int at;  // -1: none
    float t, x;
};

// returns whether an index was out of range
template <typename T, int G, int E>
__device__ __forceinline__ bool load_entries(const T* __restrict__ row, i64 r, int l, int V, const float* __restrict__ top,
                                             const int* __restrict__ index, int K, Entry (&e)[E]) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        e[i].at = -1;
        e[i].t = -INFINITY;
        if (l + i * G < K) {
            e[i].at = index[r * K + l + i * G];
            e[i].t = top[r * K + l + i * G];
        }
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        e[i].x = -INFINITY;
        if ((unsigned)e[i].at < (unsigned)V) {
            e[i].x = Elem<T>::to_f32(row[e[i].at]);
        } else {
            bad |= e[i].at != -1;
            e[i].at = -1;
            e[i].t = -INFINITY;
        }
    }
    return bad;
}

// The teacher's probabilities of a row: q of this lane's entries, their logarithms, and the mass Q of the list.
template <int G, bool TAIL, int E>
__device__ __forceinline__ void teacher(const Entry (&e)[E], const Temper& tp, float (&q)[E], float (&logq)[E], float& Q) {
    float sum = 0.f;
    if (TAIL) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            logq[i] = e[i].t;
            q[i] = fast_exp2(e[i].t * kLog2e);
            sum += q[i];
        }
        Q = row_sum<G>(sum);
        return;
    }
    float mt = -INFINITY;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        logq[i] = e[i].t;
        mt = fmaxf(mt, e[i].t);
    }
    mt = row_max<G>(mt);
    if (mt == -INFINITY) {  // an empty list, or one of -inf only (or NaN)
#pragma unroll
        for (int i = 0; i < E; ++i) {
            q[i] = logq[i] != logq[i] ? logq[i] : 0.f;
            sum += q[i];
        }
        Q = row_sum<G>(sum);
        return;
    }
    // the difference first, in 64 bits: t / T as one fp32 number is off by half a step of its own, which for values far
    // from zero or a small T is no small part of the difference
#pragma unroll
    for (int i = 0; i < E; ++i) {
        logq[i] = (float)(((double)e[i].t - (double)mt) * tp.inv);
        q[i] = fast_exp2(logq[i] * kLog2e);
        sum += q[i];
    }
    sum = row_sum<G>(sum);
    const float logs = kLn2 * log2_of_sum(sum);
#pragma unroll
    for (int i = 0; i < E; ++i) {
        q[i] /= sum;
        logq[i] -= logs;
    }
    Q = sum != sum ? sum : 1.f;
}

// e^t in 64 bits to about 1e-11, t <= 0 or moderate: t = n ln 2 + x with |x| <= ln 2 / 2, the series of e^x to
// x^9 (x^10 / 10! = 7e-12), times 2^n.  A third of the instructions of the library's exp, whose last digits
// the difference 1 - sum q does not need.
__device__ __forceinline__ double exp_f64(float t) {
    const float tc = fminf(fmaxf(t, -1000.f), 700.f);
    const double n = (double)rintf(tc * kLog2e);
    const double x = fma(n, -0.6931471805599453, (double)tc);
    double p = 1.0 / 362880.0;
    p = fma(p, x, 1.0 / 40320.0);
    p = fma(p, x, 1.0 / 5040.0);
    p = fma(p, x, 1.0 / 720.0);
    p = fma(p, x, 1.0 / 120.0);
    p = fma(p, x, 1.0 / 24.0);
    p = fma(p, x, 1.0 / 6.0);
    p = fma(p, x, 0.5);
    p = fma(p, x, 1.0);
    p = fma(p, x, 1.0);
    return t != t ? (double)t : ldexp(p, (int)n);
}

// In place of a row's log2 sum: nothing is to be learned from this row, its gradient is 0 whatever it holds.  An index
// outside the vocabulary was met, or the list is empty.
constexpr float kPoisoned = INFINITY;

// Everything behind the sums of a row, by the G lanes that share it.  o: the sums over the whole row, or with
// TAIL over the entries outside the list; first: bit i, this lane's entry i is the one of its index that counts
template <int G, bool TAIL, int E>
__device__ __forceinline__ void finish_row(i64 r, bool ok, int l, Online o, const Entry (&e)[E], unsigned first, bool bad,
                                           const Temper& tp, const DistillArgs& a) {
    const float c = tp.c;
    float q[E], logq[E], Q;
    teacher<G, TAIL, E>(e, tp, q, logq, Q);
    const Online rest = o;
    if (TAIL) {
        float mx = e[0].x;
#pragma unroll
        for (int i = 1; i < E; ++i) mx = fmaxf(mx, e[i].x);
        online_rebase(o, fmaxf(o.m, row_max<G>(mx)), c);
        const Anchor anc = anchor(o.m, c);
        float listed = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) listed += (first >> i) & 1 ? fast_exp2(measure(e[i].x, anc, c)) : 0.f;
        o.s += row_sum<G>(listed);
    }
    const bool empty = o.m == -INFINITY && !(o.s != o.s);
    // Where teacher and student nearly agree the loss is the small rest of differences of logarithms: those are
    // taken in 64 bits (an error of the row's sum itself cancels, the shares being nearly those of the teacher).
    const double l2d = empty ? 0.0 : log2_f64(o.s) - (double)ms_slip(o.m, c);
    const float l2 = (float)l2d;
    // A term is rounded to fp32 once, as it enters the sum: log p of a listed entry masked with the lowest value of its
    // type is beyond fp32 where T < 1, T^2 log p where T > 1, and q T^2 log p is neither
    float loss = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i)
        loss += q[i] == 0.f || e[i].at < 0 ? 0.f : (float)((double)q[i] * ((double)logq[i] - logprob_f64(e[i].x, o.m, l2d, tp)) * tp.sq);
    loss = row_sum<G>(loss);
    float B = empty ? 0.f : Q * fast_exp2(-(l2 + ms_slip(o.m, c)));
    if (TAIL) {
        // the mass the list leaves in 64 bits: a list that holds nearly everything leaves a small difference
        double mass = 0.0;
#pragma unroll
        for (int i = 0; i < E; ++i) mass += e[i].at >= 0 ? exp_f64(e[i].t) : 0.0;
        const double left = 1.0 - group_sum_f64<G>(mass);
        const bool has_rest = rest.m > -INFINITY || rest.s != rest.s;
        const float qr = has_rest && left > 0.0 ? (float)left : 0.f;
        B = 0.f;
        if (has_rest) {
            const double l2rd = log2_f64(rest.s) - (double)ms_slip(rest.m, c);
            const float l2r = (float)l2rd;
            if (qr > 0.f) {
                const double logpr = ((double)rest.m - (double)o.m) * tp.inv + (l2rd - l2d) * 0.6931471805599453;
                loss += (float)((double)qr * (log2_f64(qr) * 0.6931471805599453 - logpr) * tp.sq);
            }
            const float to_all = anchor_shift(rest.m, o.m, c) - (l2 + ms_slip(o.m, c));
            B = (Q + qr) * fast_exp2(to_all) - qr * fast_exp2(-(l2r + ms_slip(rest.m, c)));
        }
    }
    int seen = bad ? 2 : 0;
#pragma unroll
    for (int i = 0; i < E; ++i) seen |= e[i].at >= 0 ? 1 : 0;
    seen = group_allreduce_i32<G, OpMaxI>(seen);  // 0: an empty list, 1: entries, 2 and more: an index out of range
    bad = seen > 1;
    if (bad && a.status) raise_flag(a.status, CWR_FLAG_BAD_LABEL);
    if (!ok || l != 0) return;
    a.loss[r] = bad ? __int_as_float(0x7fc00000) : seen == 0 ? 0.f : loss;
    if (a.stat) a.stat[r] = seen != 1 ? make_float4(0.f, 0.f, 0.f, kPoisoned) : make_float4(rest.m, B, o.m, l2);
}

// G lanes per row (the row whole in registers), or one or NW waves per row that walk it in chunks.
template <typename T, int G, int E, int NW, bool TAIL, bool EDGE>
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
    Entry e[E];
    const bool bad = load_entries<T, G, E>(row, rr, l, V, a.top, a.index, a.K, e);
    unsigned first = 0;

    Online o = {-INFINITY, 0.f, 0.f};
    for (int ch = first_chunk; ch < chunks; ch += NW) {
        float v[kLaneElems];
        unpack_chunk<T>(next, v);
        mask_chunk<T, G, EDGE>(v, ch * CHUNK - off, l, V);
        if (G == 64 && ch + NW < chunks) fetch(ch + NW);
        if (TAIL) {
            marks[w][lane] = 0;
            wave_sync();
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const int place = e[i].at + off - ch * CHUNK;
                if (e[i].at >= 0 && place >= 0 && place < CHUNK) {
                    const int pk = place / VEC;
                    const unsigned bit = 1u << ((pk / G) * VEC + (place & (VEC - 1)));
                    // of entries that name one index, the one that sets the mark counts
                    if ((atomicOr(&marks[w][g * G + (pk & (G - 1))], bit) & bit) == 0) first |= 1u << i;
                }
            }
            wave_sync();
            const unsigned mine = marks[w][lane];
#pragma unroll
            for (int s = 0; s < kLaneElems; ++s) {  // bit s as a mask of all bits chooses between -inf and the value
                const int m = (int)(mine << (31 - s)) >> 31;
                v[s] = __int_as_float((m & (int)0xff800000) | (~m & __float_as_int(v[s])));
            }
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
            static_assert(NW == 1 || E == 1, "a wave has a lane for every entry");
            first = e[0].at >= 0 ? 1u : 0u;
            for (int j = 0; j < a.K; ++j)
                if (__builtin_amdgcn_readlane(e[0].at, j) == e[0].at && j < lane) first = 0;
        }
    }
    finish_row<G, TAIL, E>(r, ok, l, o, e, first, bad, tp, a);
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
template <typename T, int G, int E, bool TAIL, bool EDGE>
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
    Entry e[E];
    load_entries<T, G, E>(row, r, l, V, top, index, K, e);
    const float4 st = stat[r];
    float gt = go.p[r * go.stride] * go.scale / (float)tp.inv;
    int* map = map_[w] + g * CHUNK;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        int* p = map + (i * G + l) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) p[j] = kUnset;
    }
    float q[E], logq[E], Q;
    teacher<G, TAIL, E>(e, tp, q, logq, Q);
    if (TAIL && st.x > -INFINITY) Q = fmaxf(Q, 1.f);  // with the tail's mass, where there is a tail
    const float c = tp.c;
    const Anchor ref = anchor(st.x, c);
    const bool poisoned = st.w == kPoisoned;  // no gradient
    const float B = poisoned ? 0.f : st.y * gt;
    wave_sync();
    int place[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        place[i] = e[i].at >= 0 && e[i].at >= e0 && e[i].at - e0 < CHUNK ? e[i].at - e0 : -1;
        if (place[i] >= 0) map[place[i]] = l + i * G;
    }
    wave_sync();
    bool twice = false;
#pragma unroll
    for (int i = 0; i < E; ++i) twice |= place[i] >= 0 && map[place[i]] != l + i * G;
    if (__ballot(twice) != 0) {  // an index listed more than once: its shares add up, in the list's order
        float sum[E];
#pragma unroll
        for (int i = 0; i < E; ++i) sum[i] = 0.f;
#pragma unroll
        for (int k = 0; k < E; ++k)
            for (int j = 0; j < G; ++j) {
                const float qj = __shfl(q[k], g * G + j);
                const int aj = __shfl(e[k].at, g * G + j);
#pragma unroll
                for (int i = 0; i < E; ++i) sum[i] += aj == e[i].at ? qj : 0.f;
            }
#pragma unroll
        for (int i = 0; i < E; ++i) q[i] = sum[i];
    }
    wave_sync();
    const bool empty = st.z == -INFINITY && st.w == st.w;
    const Anchor anc = anchor(st.z, c);
    const float total = st.w + ms_slip(st.z, c);
#pragma unroll
    for (int i = 0; i < E; ++i)
        if (place[i] >= 0) {
            const float p = empty ? 0.f : fast_exp2(measure(e[i].x, anc, c) - total);
            map[place[i]] = poisoned ? 0 : __float_as_int(gt * fmaf(p, Q, -q[i]));
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
// Lanes per row: enough for the row, 16 elements each, and for its list, four entries each (a lane per entry
// widened the group of a short row: 1022684 rows of 102 fp16 entries with lists of 34 took 1100 us, forward
// and backward, with one row per wave).
static int list_group(int span, int K) {
    int G = 4;
    while (G < 64 && (G * kLaneElems < span || 4 * G < K)) G *= 2;
    return G;
}

template <typename T, bool TAIL, bool EDGE>
static int distill_typed(const T* x, i64 R, int V, i64 stride, const Temper& tp, const DistillArgs& a,
                         hipStream_t stream) {
    const int span = V + (EDGE ? RowPacks<T>::VEC - 1 : 0);  // places a row can take on the pack grid
    const int G = list_group(span, a.K);
#define CWR_GROUP_E(GG, EE)                                                                                         \
    {                                                                                                               \
        const i64 waves = (R + 64 / GG - 1) / (64 / GG);                                                            \
        if (waves > kMaxWaves) return CWR_ERR_TOO_LARGE;                                        \
        CWR_LAUNCH((k_distill<T, GG, EE, 1, TAIL, EDGE>), dim3(wave_blocks(waves)), dim3(kWavesPerBlock * 64), 0,   \
                   stream, x, R, V, stride, tp, a);                                                                 \
        return check_launch();                                                                                      \
    }
#define CWR_GROUP(GG)                                                                                               \
    if (G == GG) {                                                                                                  \
        if (a.K <= GG) CWR_GROUP_E(GG, 1)                                                                           \
        CWR_GROUP_E(GG, 4)                                                                                          \
    }
    CWR_GROUP(4) CWR_GROUP(8) CWR_GROUP(16) CWR_GROUP(32)
#undef CWR_GROUP
    const i64 chunks = ((i64)span + 64 * kLaneElems - 1) / (64 * kLaneElems);
    const int NW = row_waves(R, chunks);
    if (R > kMaxWaves) return CWR_ERR_TOO_LARGE;
    if (NW == 1) CWR_GROUP_E(64, 1)
#undef CWR_GROUP_E
    if (NW == 16)
        CWR_LAUNCH((k_distill<T, 64, 1, 16, TAIL, EDGE>), dim3((unsigned)R), dim3(1024), 0, stream, x, R, V, stride, tp, a);
    else
        CWR_LAUNCH((k_distill<T, 64, 1, 4, TAIL, EDGE>), dim3((unsigned)R), dim3(256), 0, stream, x, R, V, stride, tp, a);
    return check_launch();
}

template <typename T, bool TAIL, bool EDGE>
static int distill_grad_typed(const T* x, i64 R, int V, i64 stride, const Temper& tp, const RowDistill& s, const GradOut& go,
                              T* dx, hipStream_t stream) {
    const int span = V + (EDGE ? RowPacks<T>::VEC - 1 : 0);
    const int G = list_group(span, (int)s.K);
    const i64 chunks = G < 64 ? 1 : ((i64)span + 64 * kLaneElems - 1) / (64 * kLaneElems);
    const i64 waves = G < 64 ? (R + 64 / G - 1) / (64 / G) : R * chunks;
    if (waves > kMaxWaves) return CWR_ERR_TOO_LARGE;
#define CWR_GROUP_E(GG, EE)                                                                                              \
    {                                                                                                                    \
        CWR_LAUNCH((k_distill_grad<T, GG, EE, TAIL, EDGE>), dim3(wave_blocks(waves)), dim3(kWavesPerBlock * 64), 0,      \
                   stream, x, R, V, stride, tp, s.top, s.index, (int)s.K, reinterpret_cast<const float4*>(s.stat), go,   \
                   (int)chunks, dx);                                                                                     \
        return check_launch();                                                                                           \
    }
#define CWR_GROUP(GG)                                                                                                    \
    if (G == GG) {                                                                                                       \
        if (s.K <= GG) CWR_GROUP_E(GG, 1)                                                                                \
        CWR_GROUP_E(GG, 4)                                                                                               \
    }
    CWR_GROUP(4) CWR_GROUP(8) CWR_GROUP(16) CWR_GROUP(32)
    CWR_GROUP_E(64, 1)
#undef CWR_GROUP
#undef CWR_GROUP_E
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
