// Scores of the rows of a logit tensor: log-probabilities of given tokens, the entropy and the most
// probable entries of softmax(x / T) per row, and the gradient of all three.
//
//   forward   z = x / T, lse = log sum exp z;  log p_i = z_i - lse;  H = -sum p log p = lse - sum p z;
//             the K largest entries, equal ones by ascending index.
//   backward  with w_i the gradient that arrives at log p_i (given tokens and alternatives alike), W their
//             sum, g_H and g_lse those of the entropy and of lse:
//             dx_v = (1/T) [ sum_{i = v} w_i - p_v (W - g_lse + g_H (log p_v + H)) ].
//
// The reference has no counterpart (its callers run log_softmax on stored logits, test/test.py:19-20).
//
// Bound: HBM.  The forward pass reads every logit once, the backward pass reads it once more and
// writes its gradient; everything else is a few dozen bytes a row.
#include "cwr_host.hpp"
#include "cwr_rowwalk.hpp"

namespace cwr {

struct ScoreArgs {
    const int* tokens;  // (R, M)
    int M, K;
    float4* stat;  // (R) maximum, log2 of the sum of 2^((x - max) c), entropy, 0; may be null
    float* logprobs;
    float* entropy;
    float* lse;
    float* top_logprobs;
    int* top_index;
    int* status;  // may be null
};

// The given tokens of a row, one per lane of the G lanes that share it (and round), in two steps: their
// logits are asked for along with the row itself, so that nothing waits for them at the end.
struct TokenLogit {
    int tok;
    float x;
};
__device__ __forceinline__ TokenLogit fetch_token_index(i64 r, int j, const ScoreArgs& a) {
    TokenLogit t = {-1, 0.f};
    if (j < a.M) t.tok = a.tokens[r * a.M + j];
    return t;
}
template <typename T>
__device__ __forceinline__ void fetch_token_logit(TokenLogit& t, const T* __restrict__ row, int V) {
    if ((unsigned)t.tok < (unsigned)V) t.x = Elem<T>::to_f32(row[t.tok]);
}

__device__ __forceinline__ void write_token(const TokenLogit& t, float lp, i64 r, int j, int V, const ScoreArgs& a) {
    if (j >= a.M) return;
    if ((unsigned)t.tok >= (unsigned)V) {
        lp = 0.f;  // -1: no token
        if (t.tok != -1) {
            lp = __int_as_float(0x7fc00000);
            if (a.status) raise_flag(a.status, CWR_FLAG_BAD_LABEL);
        }
    }
    a.logprobs[r * a.M + j] = lp;
}

// maximum m, l2 = log2_sum, o the row's sums: what is known of the row as a whole
__device__ __forceinline__ void write_row(i64 r, const Online& o, float l2, const Temper& tp, const ScoreArgs& a) {
    const bool empty = o.m == -INFINITY;  // nothing but -inf
    if (a.lse) a.lse[r] = empty ? (l2 != l2 ? l2 : -INFINITY)
                                : (float)((double)o.m * tp.inv + (double)l2 * 0.6931471805599453);
    // H = -sum p ln p with log2 p = t - log2(s): the slip of ms is in both and cancels
    const float h = empty ? (l2 != l2 ? l2 : 0.f) : kLn2 * (log2_of_sum(o.s) - o.u / o.s);
    if (a.entropy) a.entropy[r] = h;
    if (a.stat) a.stat[r] = make_float4(o.m, l2, h, 0.f);
}

// log2_sum with the empty row's answer
__device__ __forceinline__ float row_l2(const Online& o, float c) {
    return o.m == -INFINITY && !(o.s != o.s) ? 0.f : log2_sum(o, c);
}

// ---------------------------------------------------------------------------------------------
// ranking
// ---------------------------------------------------------------------------------------------
// Floats as integers of the same order; -0 counts as +0, so that the two tie as they do as numbers.
__device__ __forceinline__ int order_i32(float f) {
    const int b = __float_as_int(f + 0.f);
    return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float from_order_i32(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }

// ---------------------------------------------------------------------------------------------
// G = 4 .. 32 lanes per row, the row whole in registers
// ---------------------------------------------------------------------------------------------
// Alternatives one after the other: every lane scans its 16 values for its best, the group agrees on
// the best of those (ties by index) and its owner strikes it out.  About 95 instructions a round and
// wave, shared by 64 / G rows.
template <typename T, int G, bool EDGE>
__global__ __launch_bounds__(kWavesPerBlock * 64) void k_scores_group(const T* __restrict__ x, i64 R, int V, i64 stride,
                                                                      const Temper tp, const ScoreArgs a) {
    constexpr int VEC = RowPacks<T>::VEC, NP = RowPacks<T>::NP, RP = 64 / G;
    const int lane = threadIdx.x & 63, l = lane & (G - 1);
    const i64 r = wave_first_row<true>(RP) + lane / G;
    if (r - lane / G >= R) return;
    const bool ok = r < R;
    const T* row = x + (ok ? r : R - 1) * stride;
    const int off = EDGE ? grid_offset(row) : 0;
    TokenLogit tok = fetch_token_index(ok ? r : R - 1, l, a);
    v4i raw[NP];
    load_chunk<T, G, EDGE, true>(row, -off, l, V, raw);
    fetch_token_logit<T>(tok, row, V);
    float v[kLaneElems];
    unpack_chunk<T>(raw, v);
    mask_chunk<T, G, EDGE>(v, -off, l, V);
    Online o;
    o.m = row_max<G>(chunk_max(v));
    online_chunk<true>(v, o.m, tp.c, o.s, o.u);
    o.s = row_sum<G>(o.s);
    o.u = row_sum<G>(o.u);
    const float l2 = row_l2(o, tp.c);
    if (ok && l == 0) write_row(r, o, l2, tp, a);
    if (ok) {
        write_token(tok, logprob(tok.x, o.m, l2, tp), r, l, V, a);
        for (int j = l + G; j < a.M; j += G) {
            TokenLogit more = fetch_token_index(r, j, a);
            fetch_token_logit<T>(more, row, V);
            write_token(more, logprob(more.x, o.m, l2, tp), r, j, V, a);
        }
    }
    if (a.K == 0) return;
    int key[kLaneElems];
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const int e = (i * G + l) * VEC - off + j;
            // NaN ranks as -inf; what lies outside the row ranks below everything
            key[i * VEC + j] = (unsigned)e < (unsigned)V ? order_i32(fmaxf(v[i * VEC + j], -INFINITY)) : INT_MIN;
        }
    int out_key = 0, out_idx = 0;
    for (int k = 0; k < a.K; ++k) {
        int best = key[0], slot = 0;
#pragma unroll
        for (int s = 1; s < kLaneElems; ++s) {
            const bool more = key[s] > best;
            best = more ? key[s] : best;
            slot = more ? s : slot;
        }
        const int e = ((slot / VEC) * G + l) * VEC + (slot & (VEC - 1)) - off;
        const int top = group_allreduce_i32<G, OpMaxI>(best);
        const int at = group_allreduce_i32<G, OpMinI>(best == top ? e : INT_MAX);
        const int strike = best == top && e == at ? slot : -1;
#pragma unroll
        for (int s = 0; s < kLaneElems; ++s) key[s] = s == strike ? INT_MIN : key[s];
        if ((k & (G - 1)) == l) {
            out_key = top;
            out_idx = at;
        }
        if ((k & (G - 1)) == G - 1 || k == a.K - 1) {  // lane l holds alternative number (k / G) G + l
            const int mine = (k & ~(G - 1)) + l;
            if (ok && mine <= k) {
                a.top_index[r * a.K + mine] = out_idx;
                a.top_logprobs[r * a.K + mine] = logprob(from_order_i32(out_key), o.m, l2, tp);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------
// one wave, or NW waves, per row
// ---------------------------------------------------------------------------------------------
// Candidates for the alternatives are kept as 64-bit keys, (order of the value, ~index), in a list of
// LDS per wave: larger key = better alternative, no two alike.  A chunk adds what is at least as good as
// the worst alternative so far.  Before there are K, the bound comes from the lanes' own maxima: K of them
// are at least their K-th largest, so K entries of the row are, and in rows of random order few more
// (16 values a lane: 9 candidates on average for K = 8).  That costs 16 compares and about ten ballots a
// row where one round of striking out (above) costs a hundred instructions per alternative.
constexpr int kListCap = 128;

__device__ __forceinline__ u64 key_of(float f, int e) {
    const unsigned o = (unsigned)order_i32(f) ^ 0x80000000u;
    return ((u64)o << 32) | (u64)(0xffffffffu - (unsigned)e);
}
__device__ __forceinline__ float key_value(u64 k) { return from_order_i32((int)((unsigned)(k >> 32) ^ 0x80000000u)); }
__device__ __forceinline__ int key_index(u64 k) { return (int)(0xffffffffu - (unsigned)(k & 0xffffffffu)); }

// The best min(n, K) of the n keys of a wave's list, sorted, in its first places.  Returns how many.
__device__ __forceinline__ int list_compress(u64* list, int n, int K) {
    const int lane = threadIdx.x & 63;
    const u64 a = lane < n ? list[lane] : 0;
    int ra = 0;
    if (n <= 64) {
#pragma unroll 2
        for (int c = 0; c < n; ++c) ra += list[c] > a ? 1 : 0;
        wave_sync();
        if (lane < n && ra < K) list[ra] = a;
    } else {
        const u64 b = lane + 64 < n ? list[lane + 64] : 0;
        int rb = 0;
#pragma unroll 2
        for (int c = 0; c < n; ++c) {
            const u64 other = list[c];
            ra += other > a ? 1 : 0;
            rb += other > b ? 1 : 0;
        }
        wave_sync();
        if (ra < K) list[ra] = a;
        if (lane + 64 < n && rb < K) list[rb] = b;
    }
    wave_sync();
    return n < K ? n : K;
}

// Largest bound found in a few steps that at least K of the lanes' values reach (as order_i32).  `top` is the
// largest of them.  One compare per step on the vector unit, the search itself on the scalar unit.
__device__ __forceinline__ int kth_bound(float lane_best, float top, int K) {
    const int mine = order_i32(lane_best);
    int lo = __builtin_amdgcn_readfirstlane(order_i32(wave_min(lane_best)));
    // the bound lies in [lo, lo + span]
    unsigned span = (unsigned)__builtin_amdgcn_readfirstlane(order_i32(top)) - (unsigned)lo;
    for (int step = 0; step < 20 && span > 0; ++step) {
        const unsigned half = (span + 1) >> 1;
        const int mid = (int)((unsigned)lo + half);
        const int reach = __popcll(__ballot(mine >= mid));
        if (reach >= K) {
            lo = mid;
            span -= half;
            if (reach == K) break;
        } else {
            span = half - 1;
        }
    }
    return lo;
}

struct Ranking {
    u64* list;
    int n;
    u64 bound;   // keys have to lie above it
    float floor_;  // the value in it
};

// Adds one value per lane (row element e, inside the row where `in`) to the list.
__device__ __forceinline__ void rank_append(Ranking& q, float f, int e, bool in) {
    const u64 key = key_of(f, e);
    const bool take = in && key > q.bound;
    const u64 takers = __ballot(take);
    if (take) q.list[q.n + __popcll(takers & ((1ull << (threadIdx.x & 63)) - 1))] = key;
    q.n += __popcll(takers);
}

// Cuts the list back to its best K and raises the bound to the last of them.
__device__ __forceinline__ void rank_tighten(Ranking& q, int K) {
    q.n = list_compress(q.list, q.n, K);
    if (q.n == K) {
        q.bound = q.list[K - 1];
        q.floor_ = key_value(q.bound);
    }
}

// v[s] for a slot that differs between the lanes: selects of values (a choice between elements of the
// array itself would put the array into memory)
__device__ __forceinline__ float pick(bool second, float x, float y) { return second ? y : x; }
__device__ __forceinline__ float pick16(const float (&v)[kLaneElems], unsigned s) {
    const bool s1 = s & 1, s2 = s & 2, s4 = s & 4, s8 = s & 8;
    const float b0 = pick(s2, pick(s1, v[0], v[1]), pick(s1, v[2], v[3]));
    const float b1 = pick(s2, pick(s1, v[4], v[5]), pick(s1, v[6], v[7]));
    const float b2 = pick(s2, pick(s1, v[8], v[9]), pick(s1, v[10], v[11]));
    const float b3 = pick(s2, pick(s1, v[12], v[13]), pick(s1, v[14], v[15]));
    return pick(s8, pick(s4, b0, b1), pick(s4, b2, b3));
}

// Bit s: v[s] >= bound (and, above the largest finite number, more).  The sign of v - bound is shifted in, two
// instructions a value and no scalar register between them: a vector instruction may read one that another vector
// instruction wrote (a compare's result as a carry) only two wait states later.  The bound is the wave's and its
// exceptions are settled on the scalar unit: zero is taken as -0, so that -0 - bound is +0; everything reaches
// -inf, and +inf is let in by the largest finite number (the difference of two infinities has no sign).
__device__ __forceinline__ unsigned reach_mask(const float (&v)[kLaneElems], float bound) {
    constexpr unsigned all = (1u << kLaneElems) - 1;
    const int bits = __builtin_amdgcn_readfirstlane(__float_as_int(bound));
    if (bits == (int)0xff800000) return all;
    const float f = __int_as_float(bits == 0 ? (int)0x80000000 : bits == 0x7f800000 ? 0x7f7fffff : bits);
    unsigned below = 0;
#pragma unroll
    for (int s = kLaneElems - 1; s >= 0; --s) below = __builtin_amdgcn_alignbit(below, (unsigned)__float_as_int(v[s] - f), 31);
    return ~below & all;
}

template <int VEC>
__device__ __forceinline__ void rank_chunk(Ranking& q, const float (&v)[kLaneElems], float best, int e0, int V, int K) {
    if (__ballot(best >= q.floor_) == 0) return;
    // every lane notes which of its values reach the bound; all lanes then hand in one of them at a time
    // (about one lane in eight has any, hardly one has two)
    unsigned reach = reach_mask(v, q.floor_);
    for (;;) {
        const u64 some = __ballot(reach != 0);
        if (some == 0) break;
        // many equal or many rising values: the list is cut back, and the bound raised, as often as it fills up
        if (q.n + __popcll(some) > kListCap) rank_tighten(q, K);
        const unsigned s = (unsigned)(__ffs((int)reach) - 1) & 15u;  // (none left: any)
        const float f = pick16(v, s);
        const int e = e0 + (int)((s / VEC) * 64 * VEC + (s & (VEC - 1)));
        rank_append(q, f, e, reach != 0 && (unsigned)e < (unsigned)V);
        reach &= reach - 1;
        wave_sync();
    }
}

template <typename T, int NW, bool EDGE>
__global__ __launch_bounds__(64 * (NW > 1 ? NW : kWavesPerBlock), sizeof(T) == 2 ? 8 : sizeof(T) == 4 ? 6 : 4) void k_scores_wave(
    const T* __restrict__ x, i64 R, int V, i64 stride, const Temper tp, const ScoreArgs a) {
    constexpr int VEC = RowPacks<T>::VEC, NP = RowPacks<T>::NP;
    constexpr int WB = NW > 1 ? NW : kWavesPerBlock;
    constexpr int CHUNK = 64 * kLaneElems;
    __shared__ u64 lists[WB][kListCap];
    __shared__ Online parts[WB];
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const i64 r = NW > 1 ? (i64)blockIdx.x : wave_first_row<true>(1);
    if (r >= R) return;  // NW > 1: one workgroup per row, none beyond
    const T* row = x + r * stride;
    const int off = EDGE ? grid_offset(row) : 0;
    const int first = NW > 1 ? w : 0;  // chunks first, first + NW, ...
    const int chunks = (int)(((i64)V + off + CHUNK - 1) / CHUNK);

    Online o = {-INFINITY, 0.f, 0.f};
    Ranking q = {lists[w], 0, 0, -INFINITY};
    v4i next[NP];
    auto fetch = [&](int ch) { load_chunk<T, 64, EDGE, true>(row, ch * CHUNK - off, lane, V, next); };
    TokenLogit tok = fetch_token_index(r, lane, a);
    if (first < chunks) fetch(first);
    fetch_token_logit<T>(tok, row, V);
    for (int ch = first; ch < chunks; ch += NW) {
        float v[kLaneElems];
        unpack_chunk<T>(next, v);
        mask_chunk<T, 64, EDGE>(v, ch * CHUNK - off, lane, V);
        if (ch + NW < chunks) fetch(ch + NW);
        float best = chunk_max(v);
        const float top = wave_max(best);
        online_rebase(o, fmaxf(o.m, top), tp.c);
        float s, u;
        online_chunk<true>(v, o.m, tp.c, s, u);
        o.s += s;
        o.u += u;
        if (a.K == 0) continue;
        if (__ballot(s != s) != 0) {  // NaN (or +inf) in the chunk: NaN ranks as -inf
#pragma unroll
            for (int i = 0; i < kLaneElems; ++i) v[i] = fmaxf(v[i], -INFINITY);
            best = fmaxf(best, -INFINITY);
        }
        if (ch == first) {
            const int lo = kth_bound(best, top, a.K);
            q.floor_ = from_order_i32(lo);
            q.bound = (u64)((unsigned)lo ^ 0x80000000u) << 32;  // below every key of that value
        }
        rank_chunk<VEC>(q, v, best, ch * CHUNK + lane * VEC - off, V, a.K);
        // before more chunks: a bound as tight as the list allows, or every chunk hands in as many as the first
        // (2048 rows of 50257 bf16 entries, K = 32: 79 us without)
        if (ch + NW < chunks && (ch == first || q.n > a.K + a.K / 2 + 8)) rank_tighten(q, a.K);
    }

    // the lanes' sums, then the waves'
    o.s = wave_sum(o.s);
    o.u = wave_sum(o.u);
    if (a.K > 0) q.n = list_compress(q.list, q.n, a.K);
    if (NW > 1) {
        if (lane == 0) parts[w] = o;
        for (int k = q.n + lane; k < a.K; k += 64) q.list[k] = 0;  // places without an entry: below every key
        __syncthreads();
        if (w == 0) {
            float m = parts[0].m;
#pragma unroll
            for (int i = 1; i < NW; ++i) m = fmaxf(m, parts[i].m);
            online_rebase(o, m, tp.c);
#pragma unroll
            for (int i = 1; i < NW; ++i) {
                Online p = parts[i];
                online_rebase(p, m, tp.c);
                o.s += p.s;
                o.u += p.u;
            }
        }
        // two lists into one, until one is left
        if (a.K > 0) {
#pragma unroll
            for (int left = NW / 2; left >= 1; left /= 2) {
                u64 mine[2];
#pragma unroll
                for (int s = 0; s < 2; ++s) mine[s] = w < left && lane < a.K ? lists[2 * w + s][lane] : 0;
                __syncthreads();
                if (w < left) {
#pragma unroll
                    for (int s = 0; s < 2; ++s)
                        if (lane < a.K) q.list[s * a.K + lane] = mine[s];
                    wave_sync();
                    list_compress(q.list, 2 * a.K, a.K);
                }
                __syncthreads();
            }
        }
        if (w != 0) return;
    }
    const float l2 = row_l2(o, tp.c);
    if (lane == 0) write_row(r, o, l2, tp, a);
    if (a.M <= 32 && a.K <= 32) {  // one logarithm for both: tokens in the lower half of the wave, alternatives above
        const int k = lane - 32;
        const u64 key = k >= 0 && k < a.K ? q.list[k] : 0;
        const TokenLogit both = {tok.tok, lane < 32 ? tok.x : key_value(key)};
        const float lp = logprob(both.x, o.m, l2, tp);
        if (lane < 32) write_token(both, lp, r, lane, V, a);
        else if (k < a.K) {
            a.top_index[r * a.K + k] = key_index(key);
            a.top_logprobs[r * a.K + k] = lp;
        }
        return;
    }
    write_token(tok, logprob(tok.x, o.m, l2, tp), r, lane, V, a);
    if (lane < a.K) {
        const u64 key = q.list[lane];
        a.top_index[r * a.K + lane] = key_index(key);
        a.top_logprobs[r * a.K + lane] = logprob(key_value(key), o.m, l2, tp);
    }
}

// ---------------------------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------------------------
struct ScoreGrads {
    const float4* stat;
    const int* tokens;
    const int* top_index;
    int M, K;
    const float* g_logprobs;  // each may be null
    const float* g_entropy;
    const float* g_lse;
    const float* g_top;
};

constexpr int kMaxEntries = 128;  // given tokens + alternatives of a row
constexpr int kUnset = 0x7fedcba9;  // a NaN no arithmetic here produces: no entry of this row

// One wave per chunk of a row (G = 64) or per 64 / G whole rows.  The gradient of every entry is
// 2^t (k1 t + k0) with two numbers per row; the few entries that are given tokens or alternatives have
// their gradient worked out by one lane each, put into a map of the chunk in LDS, and are picked up
// from there, so that every element is written exactly once and entries named twice are summed in a
// fixed order.
template <typename T, int G, bool EDGE>
__global__ __launch_bounds__(kWavesPerBlock * 64) void k_scores_grad(const T* __restrict__ x, i64 R, int V, i64 stride,
                                                                     const Temper tp, const ScoreGrads a,
                                                                     int chunks_per_row, T* __restrict__ dx) {
    constexpr int VEC = RowPacks<T>::VEC, NP = RowPacks<T>::NP, RP = 64 / G;
    constexpr int CHUNK = G * kLaneElems, ENT = kMaxEntries / RP;
    __shared__ __attribute__((aligned(16))) int map_[kWavesPerBlock][64 * kLaneElems];
    __shared__ int ent_idx[kWavesPerBlock][kMaxEntries];
    __shared__ float ent_g[kWavesPerBlock][kMaxEntries];
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
    load_chunk<T, G, EDGE, true>(row, e0, l, V, raw);

    // the row's entries and their incoming gradients
    const int n = a.M + a.K;
    int* map = map_[w] + g * CHUNK;
    int* idx = ent_idx[w] + g * ENT;
    float* gin = ent_g[w] + g * ENT;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        int* p = map + (i * G + l) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) p[j] = kUnset;
    }
    int my_idx[2];
    float wsum = 0.f;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const int e = l + s * G;
        int at = -1;
        float gr = 0.f;
        if (e < a.M) {
            at = a.tokens[r * a.M + e];
            if (a.g_logprobs) gr = a.g_logprobs[r * a.M + e];
        } else if (e < n) {
            at = a.top_index[r * a.K + e - a.M];
            if (a.g_top) gr = a.g_top[r * a.K + e - a.M];
        }
        if ((unsigned)at >= (unsigned)V) {  // no token, or one outside the vocabulary: no gradient
            at = -1;
            gr = 0.f;
        }
        my_idx[s] = at;
        wsum += gr;
        if (e < n) {
            idx[e] = at;
            gin[e] = gr;
        }
    }
    wsum = row_sum<G>(wsum);

    const float4 st = a.stat[r];
    const float m = st.x, l2 = st.y;
    const bool empty = m == -INFINITY && l2 == l2;  // NaN rows stay NaN
    const Anchor anc = anchor(m, tp.c);
    const float slip = ms_slip(m, tp.c);
    // p = 2^(t - l2 - slip) = 2^t rs
    const float inv = (float)tp.inv;
    const float rs = empty ? 0.f : fast_exp2(-(l2 + slip)) * inv;
    const float gl = a.g_lse ? a.g_lse[r] : 0.f;
    float k1 = 0.f, k0 = -(wsum - gl);
    if (a.g_entropy) {
        const float gh = a.g_entropy[r];
        k1 = -gh * kLn2;
        k0 -= gh * (st.z - kLn2 * (l2 + slip));
    }
    k1 *= rs;
    k0 *= rs;
    wave_sync();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const int at = my_idx[s];
        const int place = at - e0;
        if (at >= 0 && place >= 0 && place < CHUNK) {
            float sum = 0.f;
            for (int j = 0; j < n; ++j) sum += idx[j] == at ? gin[j] : 0.f;
            const float t = measure(Elem<T>::to_f32(row[at]), anc, tp.c);
            const float d = fmaf(fast_exp2(t), fmaf(fmaxf(t, kTFloor), k1, k0), sum * inv);
            map[place] = empty ? 0 : __float_as_int(d);
        }
    }
    wave_sync();

#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int p0 = (i * G + l) * VEC, e = e0 + p0;
        float v[VEC], d[VEC];
        Pack<T>::unpack(raw[i], v);
        subtract_far(v, anc);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float t = fmaf(v[j], tp.c, -anc.ms);
            const float dense = fast_exp2(t) * fmaf(fmaxf(t, kTFloor), k1, k0);
            const int given = map[p0 + j];
            d[j] = given == kUnset ? dense : __int_as_float(given);
        }
        if (!ok || e >= V) continue;
        if (!EDGE || (e >= 0 && e + VEC <= V)) {
            store_raw<G == 64 || (!EDGE && G >= 8)>(out + e, Pack<T>::pack(d));
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if ((unsigned)(e + j) < (unsigned)V) out[e + j] = Elem<T>::from_f32(d[j]);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------
template <typename T, bool EDGE>
static int scores_typed(const T* x, i64 R, int V, i64 stride, const Temper& tp, const ScoreArgs& a, hipStream_t stream) {
    const int span = V + (EDGE ? RowPacks<T>::VEC - 1 : 0);  // places a row can take on the pack grid
    int G = 4;
    while (G < 64 && G * kLaneElems < span) G *= 2;
    // Striking out costs K rounds of every 64 / G rows, the list a fixed price per row and more from some 20
    // alternatives on, where its bound lets many in.  us per 200000 fp32 rows, struck out / listed: V = 64 (G = 4) K = 4
    // 19 / 160, K = 64 141 / 360; V = 128 (8) K = 40 172 / 479, K = 64 264 / 606; V = 256 (16) K = 20 186 / 190, K = 32
    // 277 / 207; V = 512 (32) K = 4 121 / 147, K = 8 180 / 156, K = 10 211 / 160, K = 16 301 / 170; bf16 alike.
    if (G < 64 && a.K * G > 320) G = 64;
#define CWR_GROUP(GG)                                                                                              \
    if (G == GG) {                                                                                                 \
        const i64 waves = (R + 64 / GG - 1) / (64 / GG);                                                           \
        if (waves > kMaxWaves) return CWR_ERR_TOO_LARGE;                                       \
        CWR_LAUNCH((k_scores_group<T, GG, EDGE>), dim3(wave_blocks(waves)), dim3(kWavesPerBlock * 64), 0, stream, x, \
                   R, V, stride, tp, a);                                                                           \
        return check_launch();                                                                                     \
    }
    CWR_GROUP(4) CWR_GROUP(8) CWR_GROUP(16) CWR_GROUP(32)
#undef CWR_GROUP
    const i64 chunks = ((i64)span + 64 * kLaneElems - 1) / (64 * kLaneElems);
    const int NW = row_waves(R, chunks);
    if (R > kMaxWaves) return CWR_ERR_TOO_LARGE;
    if (NW == 16)
        CWR_LAUNCH((k_scores_wave<T, 16, EDGE>), dim3((unsigned)R), dim3(1024), 0, stream, x, R, V, stride, tp, a);
    else if (NW == 4)
        CWR_LAUNCH((k_scores_wave<T, 4, EDGE>), dim3((unsigned)R), dim3(256), 0, stream, x, R, V, stride, tp, a);
    else
        CWR_LAUNCH((k_scores_wave<T, 1, EDGE>), dim3(wave_blocks(R)), dim3(kWavesPerBlock * 64), 0, stream, x, R, V,
                   stride, tp, a);
    return check_launch();
}

template <typename T, bool EDGE>
static int scores_grad_typed(const T* x, i64 R, int V, i64 stride, const Temper& tp, const ScoreGrads& a, T* dx,
                             hipStream_t stream) {
    const int span = V + (EDGE ? RowPacks<T>::VEC - 1 : 0);
    const int n = a.M + a.K;
    int G = 4;
    while (G < 64 && (G * kLaneElems < span || 2 * G < n)) G *= 2;  // two entries a lane at most
    const i64 chunks = G < 64 ? 1 : ((i64)span + 64 * kLaneElems - 1) / (64 * kLaneElems);
    const i64 waves = G < 64 ? (R + 64 / G - 1) / (64 / G) : R * chunks;
    if (waves > kMaxWaves) return CWR_ERR_TOO_LARGE;
#define CWR_GROUP(GG)                                                                                               \
    if (G == GG)                                                                                                    \
        CWR_LAUNCH((k_scores_grad<T, GG, EDGE>), dim3(wave_blocks(waves)), dim3(kWavesPerBlock * 64), 0, stream, x, \
                   R, V, stride, tp, a, (int)chunks, dx);
    CWR_GROUP(4) CWR_GROUP(8) CWR_GROUP(16) CWR_GROUP(32) CWR_GROUP(64)
#undef CWR_GROUP
    return check_launch();
}

template <typename T>
static int scores_any(const void* x, i64 R, int V, i64 stride, const Temper& tp, const ScoreArgs& a, hipStream_t stream) {
    const T* p = static_cast<const T*>(x);
    return on_grid<T>(x, stride, V) ? scores_typed<T, false>(p, R, V, stride, tp, a, stream)
                                    : scores_typed<T, true>(p, R, V, stride, tp, a, stream);
}

template <typename T>
static int scores_grad_any(const void* x, i64 R, int V, i64 stride, const Temper& tp, const ScoreGrads& a, void* dx,
                           hipStream_t stream) {
    const T* p = static_cast<const T*>(x);
    T* d = static_cast<T*>(dx);
    return on_grid<T>(x, stride, V) && on_grid<T>(dx, V, V)
               ? scores_grad_typed<T, false>(p, R, V, stride, tp, a, d, stream)
               : scores_grad_typed<T, true>(p, R, V, stride, tp, a, d, stream);
}

int launch_scores(const void* x, int dtype, i64 R, i64 V, i64 stride, double temperature, const RowScores& s,
                  hipStream_t stream) {
    if (R == 0) return CWR_OK;
    ScoreArgs a;
    a.tokens = s.tokens; a.M = (int)s.M; a.K = (int)s.K; a.stat = reinterpret_cast<float4*>(s.stat);
    a.logprobs = s.logprobs; a.entropy = s.entropy; a.lse = s.lse;
    a.top_logprobs = s.top_logprobs; a.top_index = s.top_index; a.status = s.status;
    const Temper tp = make_temper(temperature);
    switch (dtype) {
        case CWR_F32: return scores_any<float>(x, R, (int)V, stride, tp, a, stream);
        case CWR_F16: return scores_any<__half>(x, R, (int)V, stride, tp, a, stream);
        case CWR_BF16: return scores_any<bf16_t>(x, R, (int)V, stride, tp, a, stream);
        case CWR_F64: return scores_any<double>(x, R, (int)V, stride, tp, a, stream);
    }
    return CWR_ERR_DTYPE;
}

int launch_scores_grad(const void* x, int dtype, i64 R, i64 V, i64 stride, double temperature, const RowScoreGrads& s,
                       void* dx, hipStream_t stream) {
    if (R == 0) return CWR_OK;
    ScoreGrads a;
    a.stat = reinterpret_cast<const float4*>(s.stat); a.tokens = s.tokens;
    a.top_index = s.top_index; a.M = (int)s.M; a.K = (int)s.K; a.g_logprobs = s.g_logprobs;
    a.g_entropy = s.g_entropy; a.g_lse = s.g_lse; a.g_top = s.g_top;
    const Temper tp = make_temper(temperature);
    switch (dtype) {
        case CWR_F32: return scores_grad_any<float>(x, R, (int)V, stride, tp, a, dx, stream);
        case CWR_F16: return scores_grad_any<__half>(x, R, (int)V, stride, tp, a, dx, stream);
        case CWR_BF16: return scores_grad_any<bf16_t>(x, R, (int)V, stride, tp, a, dx, stream);
        case CWR_F64: return scores_grad_any<double>(x, R, (int)V, stride, tp, a, dx, stream);
    }
    return CWR_ERR_DTYPE;
}

}  // namespace cwr
