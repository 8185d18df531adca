// Attention within a window of the order: the backward pass.
//
//   dv_j = sum_i p_ij do_i            ds_ij = p_ij (do_i v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j      dk_j = scale sum_i ds_ij q_i
//   delta_i = do_i o_i                dbias[bucket] = sum of ds_ij with i - j in the bucket
//
// The weights are formed again from the scores and the forward's logarithms of
// the sums.  Two kernels, so that every sum has one owner and a fixed order
// (no atomics: results do not change from run to run): one holds 128 queries
// in registers and passes over their keys (delta, dq), the other holds 128 keys
// and passes over the queries that see them, all heads that share the key head
// in turn (dk, dv and the bias's sums by offset).  The first keys, which every
// query sees, have passes of their own for the queries beyond their window; they
// and few blocks are cut into pieces whose 32-bit sums a last kernel joins.  ds and p
// are rounded to the inputs' type for the second products, as the forward's weights
// are (in float16, those below 6e-5 keep fewer bits: gradients that small are
// scaled up by the caller's loss, as everywhere in that type); the bias's sums take
// them unrounded.
//
// Bound by the matrix products (18 D operations a pair, with the scores' second
// forming) and, as long, by their operands' reads from LDS, with the vector
// instructions of the weights between them.  Every earlier key at 2 x 4096 queries, 8
// heads of 128, bfloat16: dq 150 us, dk and dv 240, the forward 123, each as traced; a
// pass of all three takes 495 to 502 (240 billion operations of the definition, 480 to
// 486 T/s; a large library product reaches 1204).  Matrix cores and LDS are each busy for 39 and 33 % of a
// compute unit's busy cycles in dq, 33 and 34 in dk and dv (one wave a SIMD at width
// 128, two at 64).  Registers that do not fit: 6 to 16 in the key kernel of width 64
// with a bias, 5 to 12 in the query kernel of width 128 with one.
#include <algorithm>
#include <atomic>

#include "attention.hpp"

namespace pointops {
namespace attn {
namespace {

// The forward's lse is one 32-bit number.  Where a row's maximum is large (all of
// its keys carry a mask of the type's lowest value, or their scores are that large)
// the logarithm of the sum beside it is rounded, or lost altogether: exp2(s - lse)
// are then the weights but for one factor a row.  From here on a row's
// weights are added up ahead of its pass and both kernels divide by their sum; below,
// the factor lies within 2^-18 of 1 (2^-14 for the 16-bit types).
template <typename T>
__device__ __forceinline__ bool coarse(float lse) {
    const float size = __builtin_fabsf(lse);
    return size >= (sizeof(T) == 4 ? 64.f : 1024.f) && size < kInf;
}

// Gradients that are not finite are formed again pair by pair, where a product
// with a masked pair's infinity or NaN may have spread: of one query over the
// keys that it sees, and of one key over those of the rows i_from .. i_to - 1
// of a head that see it.  By a whole wave; n0 and so on are the values that a lane
// needs.
template <typename T>
__device__ __forceinline__ void careful_query(const Args& a, const Rows& grad, int b, int h, int i, int len, float lse,
                                              float delta, float share, bool n0, bool n1, T* dq) {
    const int g = h / (a.H / a.G), p = i + a.N - a.Q;
    const Seen seen = seen_by(a, p, len);
    const T* const k = a.k.at<T>(b, g);
    const T* const v = a.v.at<T>(b, g);
    CarefulPair<T> q, go, sum;
    q.load(a.q.at<T>(b, h) + i * a.q.n, a.D);
    go.load(grad.at<T>(b, h) + i * grad.n, a.D);
    const int lane = lane_id();
    n0 = n0 && lane < a.D;
    n1 = n1 && lane + kWave < a.D;
    auto settled = [&](int64_t j) {
        CarefulPair<T> kk, vv;
        const float bias = one_bias<T>(a, h, static_cast<int>(p - j));
        if (bias == -kInf) return false;
        kk.load(k + j * a.k.n, a.D);
        const float s = q.dot(kk) * a.scale_log2 + bias;
        if (s == -kInf) return false;
        vv.load(v + j * a.v.n, a.D);
        sum.add(exp2_fast(s - lse) * (go.dot(vv) - delta), kk);
        return ballot((n0 && finite(sum.x0)) || (n1 && finite(sum.x1))) == 0;
    };
    bool done = false;
    for (int j = 0; j < seen.first && !done; ++j) done = settled(j);
    for (int j = max(seen.low, seen.first); j < seen.low + seen.count && !done; ++j) done = settled(j);
    const float by = a.scale * share;
    if (n0) dq[lane] = from_float<T>(sum.x0 * by);
    if (n1) dq[lane + kWave] = from_float<T>(sum.x1 * by);
}

// A key's values that are needed.
struct Needed {
    bool k0, k1, v0, v1;
};

// Whether all that is needed has come out not finite again.
template <typename T>
__device__ __forceinline__ bool careful_key(const Args& a, const Rows& grad, const float* lse_in, const float* delta_in,
                                            const float* share_in, int b, int h, int64_t j, int i_from, int i_to, bool beyond,
                                            int len, const Needed& need, CarefulPair<T>& dk, CarefulPair<T>& dv) {
    const int g = h / (a.H / a.G);
    const int64_t stats = (static_cast<int64_t>(b) * a.H + h) * a.Q;
    auto settled = [&] {
        return ballot((need.k0 && finite(dk.x0)) || (need.k1 && finite(dk.x1)) || (need.v0 && finite(dv.x0)) ||
                      (need.v1 && finite(dv.x1))) == 0;
    };
    auto sees = [&](int64_t i) {
        const int off = static_cast<int>(i) + a.N - a.Q - static_cast<int>(j);
        return !(a.causal && off < 0) && ((off < 0 ? -off : off) < a.window) != beyond;
    };
    // A row whose lse is no number makes all of a key that it sees none, one whose delta
    // is not finite its dk: 64 rows at a time.
    bool odd_lse = false, odd_delta = false;
    for (int64_t i = i_from + lane_id(); i < i_to; i += kWave) {
        const float lse = lse_in[stats + i], delta = delta_in[stats + i];
        if ((lse == lse && finite(delta)) || lse == kInf || !sees(i)) continue;
        if (one_bias<T>(a, h, static_cast<int>(i) + a.N - a.Q - static_cast<int>(j)) == -kInf) continue;
        odd_lse |= lse != lse;
        odd_delta = true;
    }
    if (ballot(odd_delta) != 0) dk.x0 = dk.x1 = __builtin_nanf("");
    if (ballot(odd_lse) != 0) dv.x0 = dv.x1 = __builtin_nanf("");
    if (settled()) return true;
    CarefulPair<T> k, v;
    k.load(a.k.at<T>(b, g) + j * a.k.n, a.D);
    v.load(a.v.at<T>(b, g) + j * a.v.n, a.D);
    for (int64_t i = i_from; i < i_to; ++i) {
        if (!sees(i)) continue;
        const int off = static_cast<int>(i) + a.N - a.Q - static_cast<int>(j);
        const float lse = lse_in[stats + i];
        if (lse == kInf) continue;
        const float bias = one_bias<T>(a, h, off);
        if (bias == -kInf) continue;
        CarefulPair<T> q, go;
        q.load(a.q.at<T>(b, h) + i * a.q.n, a.D);
        const float s = q.dot(k) * a.scale_log2 + bias;
        if (s == -kInf) continue;
        go.load(grad.at<T>(b, h) + i * grad.n, a.D);
        const float w = exp2_fast(s - lse) * share_in[stats + i];
        dv.add(w, go);
        dk.add(w * (go.dot(v) - delta_in[stats + i]) * a.scale, q);
        if (settled()) return true;
    }
    return false;
}

// A row's output is about as large as its values where it sees few keys, and its
// rounding to 16 bits then takes as much from dq, through delta, as dq's own
// (dq's error against 64 bits at 9 x 30 queries, 6 heads of 20, float16: 1.64
// times a rounding's with it, 1.43 without).  Beyond this many keys the output is
// an average of many, and the pass over them is not made twice.  (With a bias, whose
// sums are small beside their terms, dk and the bias take delta with what the pass over
// the keys measured: `refine`, whether or not the bias's gradient is asked for.)
constexpr int kFewKeys = 128;

// A row's ds add up to zero, and in heads of few columns dq cancels the more by it: with
// ds rounded, its error is 1.45 to 1.6 times one rounding's at widths 16 to 24 (1.41 to
// 1.46 from 32 on).  There the second product is made again with what the rounding
// left (16-bit types; 1.1 times; 462 queries over 924 keys, 3 x 6 heads of 20: 23.2 ->
// 24.5 us of the kernel by queries).  Width 32 would pay 36.3 -> 44.8 us for it (4 x
// 4096 queries, 8 heads over 2, window 512).
constexpr int kNarrow = 24;

// The most keys that a row up to position p_last sees.
__device__ __forceinline__ int most_seen(const Args& a, int p_last, int len) {
    const int side = min(a.window, kFewKeys + 1), first = min(a.sinks, kFewKeys + 1);
    return a.causal ? min(side + first, p_last + 1) : min(2 * side - 1 + first, len);
}

// The sum of a wave's rows' exp2(s - lse), with the scores as the pass over the keys
// forms them; keys straight from memory, as few rows ask for it.
template <typename T, int DP, bool VEC>
__device__ __forceinline__ float exponents_sum(const Args& a, const i32x4 (&q)[Tile<T, DP>::kChunks], const T* k, const Walk& walk,
                                               const Seen& seen, const float* table, int p, int len, float lse) {
    const int lane = lane_id(), half = lane / 32;
    const float factor = table != nullptr ? 1.f : a.scale_log2;
    float sum = 0.f;
    for (int t = walk.begin(); t < walk.end; t = walk.after(t)) {
        const int row = 32 * t + lane % 32;
        f32x16 s = {};
#pragma unroll
        for (int c = 0; c < Tile<T, DP>::kChunks; ++c) {
            i32x4 key = {0, 0, 0, 0};
            if (row < len) key = load_row<T, VEC>(k + row * a.k.n, (2 * c + half) * kPerFrag<T>, a.D);
            s = mma<T>(key, q[c], s);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int j = 32 * t + 4 * half + 8 * (r / 4) + r % 4;
            const float bias = table != nullptr ? table[min(max(p - j, -a.reach), a.reach) + a.reach + kMargin] : 0.f;
            const float x = table != nullptr ? s[r] * a.scale_log2 + bias : s[r];
            if (seen(j) && bias != -kInf) sum += exp2_fast(__builtin_fmaf(x, factor, -lse));
        }
    }
    return halves_sum(sum);
}

template <typename T, int DP, bool VEC, bool BIAS, int SPLIT>
__global__ __launch_bounds__(kThreads, (sizeof(T) == 4 && DP > 64) ? 1 : 2) void attention_grad_query_kernel(
    const Args a, const T* __restrict__ out, const float* __restrict__ lse_in, const Rows grad,
    float* __restrict__ delta_out, float* __restrict__ share_out, int* __restrict__ coarse_out,
    T* __restrict__ dq_out, const bool refine) {
    using TileT = Tile<T, DP>;
    constexpr int TK = Cut<T, SPLIT>::kInnerRows, kSub = Cut<T, SPLIT>::kSub, kRows = Cut<T, SPLIT>::kRows;
    constexpr int kOut = DP / 32, kTileBytes = TK * TileT::kStride;
    constexpr bool kTight = sizeof(T) == 2 && DP == 128;  // no registers for both products' operands at once
    extern __shared__ char lds[];  // two pairs of a key and a value tile, the bias's table
    float* const table = reinterpret_cast<float*>(lds + 4 * kTileBytes);
    const int entries = bias_entries(a.reach);

    const int lane = lane_id(), half = lane / 32, wave = uniform(threadIdx.x / kWave);
    const int wave_row = 32 * (wave % (kWaves / SPLIT)), sub = wave / (kWaves / SPLIT) * kSub;  // its rows, its pieces
    const int blocks = (a.Q + kRows - 1) / kRows;
    const Place at = place(a.B * a.H, blocks);
    const int b = at.outer / a.H, h = at.outer % a.H, g = h / (a.H / a.G);
    const int i0 = folded(at.inner, blocks) * kRows;
    const int len = a.length(b), shift = a.N - a.Q;

    const int rows = min(kRows, a.Q - i0);
    const Walk walk(a, max(i0 + shift, 0), min(i0 + shift + rows, len) - 1, len, TK);

    const int w0 = i0 + wave_row + shift;
    const int w_count = min(32, i0 + rows - (i0 + wave_row));
    const int w_first = max(w0, 0), w_last = min(w0 + w_count, len) - 1;
    const bool w_any = w_first <= w_last, w_whole = w_any && w0 >= 0 && w0 + w_count <= len;
    const int row = i0 + wave_row + lane % 32, p = row + shift;
    const bool exists = row < a.Q && p >= 0 && p < len;
    const Seen seen = seen_by(a, p, len);

    const T* const k = a.k.at<T>(b, g);
    const T* const v = a.v.at<T>(b, g);
    Stage<T, DP, TK, VEC> ks, vs;
    int t = walk.begin();
    if (t < walk.end) {
        ks.load(k, a.k.n, t * TK, len, a.D);
        vs.load(v, a.v.n, t * TK, len, a.D);
    }
    const bool biased = BIAS && (VEC || a.bias != nullptr);  // rows that are not aligned have one kernel for both
    if (biased) fill_bias<T>(a, h, table, reinterpret_cast<int*>(table + entries));
    i32x4 q[TileT::kChunks], go[TileT::kChunks];
    float delta = 0.f, lse = kInf, rest = 0.f;
    const int64_t stat = (static_cast<int64_t>(b) * a.H + h) * a.Q + row;
    {
        const T* const qrow = a.q.at<T>(b, h) + row * a.q.n;
        const T* const grow = grad.at<T>(b, h) + row * grad.n;
        const T* const orow = out + ((static_cast<int64_t>(b) * a.Q + row) * a.H + h) * a.D;
#pragma unroll
        for (int c = 0; c < TileT::kChunks; ++c) {
            const int d = (2 * c + half) * kPerFrag<T>;
            q[c] = go[c] = i32x4{0, 0, 0, 0};
            if (exists) {
                q[c] = load_row<T, VEC>(qrow, d, a.D);
                go[c] = load_row<T, VEC>(grow, d, a.D);
                const i32x4 o = load_row<T, VEC>(orow, d, a.D);
#pragma unroll
                for (int e = 0; e < kPerFrag<T>; ++e) delta = __builtin_fmaf(element<T>(o, e), element<T>(go[c], e), delta);
            }
        }
        delta = halves_sum(delta);
        if (exists) lse = lse_in[stat];
    }
    if (t < walk.end) {
        ks.store(lds);
        vs.store(lds + kTileBytes);
    }
    __syncthreads();

    float share = 1.f;
    const bool any_coarse = ballot(coarse<T>(lse)) != 0;
    if (lane == 0 && row < a.Q) coarse_out[static_cast<int64_t>(b * a.H + h) * ((a.Q + 31) / 32) + row / 32] = any_coarse;
    if (any_coarse) {
        const float sum = exponents_sum<T, DP, VEC>(a, q, k, Walk(a, w_first, w_last, len, 32), seen, biased ? table : nullptr, p, len, lse);
        if (coarse<T>(lse) && sum > 0.f && sum < kInf) share = 1.f / sum;
    }
    // The weights of a row sum to 1, so that what is left of its ds is what the
    // rounded output took from delta: of few keys a pass ahead measures it.
    // (Of a row beside a place that is no number it cannot be told.)
    auto left = [](float all) { return all - all == 0.f ? all : 0.f; };
    const bool narrow = a.D <= kNarrow;
    const float factor = biased ? 1.f : a.scale_log2;
    f32x16 dq[kOut] = {};
    char* ktile = lds;
    bool ahead = sizeof(T) == 2 && most_seen(a, min(i0 + shift + rows, len) - 1, len) <= kFewKeys;
    while (t < walk.end) {
        char* const vtile = ktile + kTileBytes;
        const int j0 = t * TK;
        t = walk.after(t);
        const bool turn = ahead && t >= walk.end;
        if (turn) t = walk.begin();
        if (t < walk.end) {
            ks.load(k, a.k.n, t * TK, len, a.D);
            vs.load(v, a.v.n, t * TK, len, a.D);
        }
        const bool meets = w_any && ((j0 <= seen_high(a, w_last, len) && j0 + TK > seen_low(a, w_first)) ||
                                     j0 < seen_first(a, w_last, len));
        if (meets) {
            const bool whole = w_whole && ((j0 + TK - 1 <= seen_high(a, w_first, len) && j0 >= seen_low(a, w_last)) ||
                                           j0 + TK <= seen_first(a, w_first, len));
            const int near = w0 - j0;
            const bool far = near - (TK - 1) >= a.reach || near + 31 <= -a.reach;
#pragma unroll
            for (int u = 0; u < kSub; ++u) {
                const int own = 32 * (sub + u);  // first row of the piece
                RowFrags<T, DP> kf, vf;
                kf.load(ktile, own);
                if (!kTight) vf.load(vtile, own);
                keep_order();
                f32x16 s = kf.times(q);
                if (kTight) vf.load(vtile, own);
                const f32x16 dp = vf.times(go);
                ColumnFrags<T, DP> cf[2];  // of this chunk of keys and the next
                cf[0].load(ktile, own);
                keep_order();
                if (biased) {
                    s *= a.scale_log2;
                    if (far) {
                        s += table[near > 0 ? entries - 1 : 0];
                    } else {
                        const float* const from = table + near + lane % 32 - 4 * half - own + a.reach + kMargin;
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[r] += from[-(8 * (r / 4) + r % 4)];
                    }
                }
                float ds[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float w = exp2_fast(__builtin_fmaf(s[r], factor, -lse));
                    ds[r] = w * (dp[r] - delta);
                }
                if (!whole) {
                    const int j = j0 + own + 4 * half;
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (!seen(j + 8 * (r / 4) + r % 4)) ds[r] = 0.f;
                }
                if (refine || ahead) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) rest += ds[r];
                }
                if (ahead) continue;
                constexpr int kSteps = 16 / kPerFrag<T>;
#pragma unroll
                for (int c = 0; c < kSteps; ++c) {
                    if (c + 1 < kSteps) cf[(c + 1) % 2].load(ktile, own + (c + 1) * TileT::kRowsPerFrag);
                    keep_order();
                    const i32x4 x = as_fragment<T>(&ds[c * kPerFrag<T>]);
                    cf[c % 2].add(x, dq);
                    if (sizeof(T) == 2 && DP == 32 && narrow) {
                        float rounded[kPerFrag<T>];
#pragma unroll
                        for (int e = 0; e < kPerFrag<T>; ++e) rounded[e] = ds[c * kPerFrag<T> + e] - element<T>(x, e);
                        cf[c % 2].add(as_fragment<T>(rounded), dq);
                    }
                }
            }
        }
        ktile = ktile == lds ? lds + 2 * kTileBytes : lds;
        if (t < walk.end) {
            ks.store(ktile);
            vs.store(ktile + kTileBytes);
        }
        __syncthreads();
        if (turn) {
            ahead = false;
            float taken = halves_sum(rest);
            if constexpr (SPLIT == 2 && sizeof(T) == 2) {
                __shared__ float parts[kWaves][32];
                if (half == 0) parts[wave][lane] = taken;
                __syncthreads();
                taken = parts[wave % 2][lane % 32] + parts[wave % 2 + 2][lane % 32];
            }
            delta += left(taken) * share;
            rest = 0.f;
        }
    }

    if constexpr (SPLIT == 2) {
        float* const other = reinterpret_cast<float*>(lds) + wave % 2 * (16 * kOut + 1) * kWave;
        if (wave >= 2) {
            put_sums(other + kWave, dq);
            other[lane] = rest;
        }
        __syncthreads();
        if (wave >= 2) return;
        rest += other[lane];
        get_sums(other + kWave, dq, 1.f, 1.f);
    }
    float odd = 0.f;  // NaN where anything is not finite
#pragma unroll
    for (int d = 0; d < kOut; ++d) {
        dq[d] *= a.scale * share;
#pragma unroll
        for (int r = 0; r < 16; ++r) odd += dq[d][r] * 0.f;
    }
    // Rows that do not exist have met the tiles too, with weights of zero: 0 * inf.
    uint64_t bad = ballot(row < a.Q && odd != 0.f);
    bad = (bad | bad >> 32) & 0xffffffffu;
    T* const dst = dq_out + ((static_cast<int64_t>(b) * a.Q + row) * a.H + h) * a.D;
    if (row < a.Q) {
#pragma unroll
        for (int d = 0; d < kOut; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) store4<T, VEC>(dst, 32 * d + 8 * e + 4 * half, a.D, dq[d], 4 * e);
    }
    if (bad != 0) {
        const uint64_t odd_dq = odd_values(dq);
        __threadfence();  // what is written again comes behind the rows' stores
        while (bad != 0) {
            const int r = __builtin_ctzll(bad);
            bad &= bad - 1;
            // Where a row's own lse or delta is no number, so is every ds of its pairs, and all of dq as it lies.
            const float row_lse = i2f(readlane(f2i(lse), r)), row_delta = i2f(readlane(f2i(delta), r));
            if (row_lse != kInf && (!finite(row_lse) || !finite(row_delta))) continue;
            const int i = i0 + wave_row + r;
            careful_query<T>(a, grad, b, h, i, row_lse == kInf ? 0 : len, row_lse, row_delta, i2f(readlane(f2i(share), r)),
                             odd_value(odd_dq, r, lane), odd_value(odd_dq, r, lane + kWave),
                             dq_out + ((static_cast<int64_t>(b) * a.Q + i) * a.H + h) * a.D);
        }
    }
    if (refine) delta += left(halves_sum(rest)) * share;
    if (row < a.Q && half == 0) {
        delta_out[stat] = delta;
        share_out[stat] = share;
    }
}

// How the passes of the keys are cut.  A key block of `rows` keys passes over the
// queries within its window, in `of_rest` pieces; the queries beyond the window, which
// see the first keys alone, are passed over by groups of 32 of those, each in
// `of_first` pieces.  A key block whose sums are in more than one place writes
// 32-bit parts.
struct Pieces {
    int rows, key_blocks, of_rest;
    int groups, of_first;

    __host__ __device__ int units() const { return key_blocks * of_rest; }
    __host__ __device__ int first_units() const { return groups * of_first; }
    __host__ __device__ int first_blocks() const { return (32 * groups + rows - 1) / rows; }
    // The blocks with parts come first.
    __host__ __device__ int joined_blocks() const { return of_rest > 1 ? key_blocks : first_blocks(); }
    __host__ __device__ bool parted(int block) const { return block < joined_blocks(); }
    // Units whose parts are kept, and their floats with the groups', of one key head.
    __host__ __device__ int kept() const { return joined_blocks() * of_rest; }
    __host__ __device__ int64_t floats(int DP) const {
        return (static_cast<int64_t>(kept()) * rows + static_cast<int64_t>(first_units()) * 32) * 2 * DP;
    }
};

// Sums of ds along the diagonals of a wave's 16 x 32 piece: rows (keys) are
// written with zeros between them, so that lane x reads diagonal x - 16 of
// every row without a test; the zeros stay for the whole kernel.  (As LDS
// atomics, one an element, the sums took 125 us of 215 at 4 x 4096 queries, 8
// heads, window 512, reach 91.)
constexpr int kSkewRow = 68;
constexpr int kSkewFloats = 16 + 16 * kSkewRow;

// FIRST: the passes beyond the window.  All waves hold the same 32 keys there
// and take 32 queries each in turn; their sums are added at the end.
template <typename T, int DP, bool VEC, bool BIAS, bool FIRST, int SPLIT>
__global__ __launch_bounds__(kThreads, DP * sizeof(T) <= 128 ? 2 : 1) void attention_grad_key_kernel(
    const Args a, const float* __restrict__ lse_in, const float* __restrict__ delta_in, const float* __restrict__ share_in,
    const int* __restrict__ coarse_in, const Rows grad,
    T* __restrict__ dk_out, T* __restrict__ dv_out, float* __restrict__ part, float* __restrict__ dbias_part,
    const Pieces cut) {
    using TileT = Tile<T, DP>;
    constexpr int TQ = Cut<T, SPLIT>::kInnerRows, kSub = Cut<T, SPLIT>::kSub, kRows = Cut<T, SPLIT>::kRows;
    constexpr int kOut = DP / 32, kTileBytes = TQ * TileT::kStride;
    constexpr bool kTight = sizeof(T) == 4 ? DP == 128 : BIAS && DP == 64;  // as above
    constexpr int kSet = 2 * kTileBytes + 8 * TQ;  // a tile of queries, one of gradients, their lse and delta
    extern __shared__ char lds[];                  // two sets, then the bias's tables
    float* const table = reinterpret_cast<float*>(lds + 2 * kSet);
    const int entries = bias_entries(a.reach);
    const bool summed = BIAS && dbias_part != nullptr;
    float* const skews = table + (entries + 3) / 4 * 4;  // one a wave, then the waves' sums by offset, the edges
    float* const sums = skews + kWaves * kSkewFloats;
    int* const edges = reinterpret_cast<int*>(summed ? sums + kWaves * entries : skews);

    const int lane = lane_id(), half = lane / 32, wave = uniform(threadIdx.x / kWave);
    const int units = FIRST ? cut.first_units() : cut.units(), pieces = FIRST ? cut.of_first : cut.of_rest;
    const Place at = place(a.B * a.G, units);
    const int bg = at.outer, b = bg / a.G, g = bg % a.G;
    // A causal call's earlier keys are seen by more rows: long and short passes meet.
    const int unit = FIRST ? at.inner : units - 1 - folded(at.inner, units);
    const int piece = unit % pieces, block = unit / pieces;
    const int len = a.length(b), shift = a.N - a.Q, group = a.H / a.G;

    // This wave's keys, one a lane column; the block's.
    const int sub = wave / (kWaves / SPLIT) * kSub;  // its pieces of a tile
    const int j0 = FIRST ? 32 * block : kRows * block, w0 = FIRST ? j0 : j0 + 32 * (wave % (kWaves / SPLIT));
    const int exist = FIRST ? min(len, a.sinks) : len;
    const int w_last = min(w0 + 32, exist) - 1, j_last = FIRST ? w_last : min(j0 + kRows, exist) - 1;
    const bool w_any = w0 <= w_last;
    const int j = w0 + lane % 32;

    // Positions from which the lane's key is seen, see_low .. see_low +
    // see_count - 1, or (beyond a window on both sides) all but those.
    const bool other = FIRST && !a.causal;
    auto window_end = [&](int key) { return key > len - a.window ? len - 1 : key + a.window - 1; };  // of the keys' own
    int see_low = a.causal ? j : j - a.window + 1;
    uint32_t see_count = static_cast<uint32_t>(max(window_end(j) - see_low + 1, 0));
    if constexpr (FIRST) {
        if (a.causal) {
            see_low = window_end(j) + 1;
            see_count = j < exist ? static_cast<uint32_t>(max(len - see_low, 0)) : 0u;
        } else if (j >= exist) {
            see_low = -1;
            see_count = 0xffffffffu;
        }
    }
    // Whether any, and whether all, of the wave's keys are seen from any (all)
    // of the positions p .. p + TQ - 1.
    auto meets = [&](int p) {
        if constexpr (FIRST) return p + TQ - 1 > window_end(w0) || (other && p <= w_last - a.window);
        return p <= window_end(w_last) && p + TQ > (a.causal ? w0 : w0 - a.window + 1);
    };
    auto wholly = [&](int p) {
        if constexpr (FIRST) return w_last == w0 + 31 && (p > window_end(w_last) || (other && p + TQ - 1 <= w0 - a.window));
        return p >= (a.causal ? w_last : w_last - a.window + 1) && p + TQ - 1 <= window_end(w0);
    };

    // Queries that see any of the block's keys, by row; tiles count from the
    // first row that exists.
    const int i_low = max(-shift, 0), i_high = min(a.Q, len - shift);
    int i_first = 0, i_last = -1;
    if (j0 <= j_last) {
        int p_low = a.causal ? j0 : j0 - a.window + 1, p_high = window_end(j_last);
        if constexpr (FIRST) {
            p_low = a.causal ? window_end(j0) + 1 : 0;
            p_high = len - 1;
        }
        i_first = max(max(p_low, 0) - shift, i_low);
        i_last = min(min(p_high, len - 1) - shift, i_high - 1);
    }
    // Their tiles, for every head in turn; this piece's share of them all.
    const int t_first = (i_first - i_low) / TQ, tiles = i_last < i_first ? 0 : (i_last - i_low) / TQ + 1 - t_first;
    const int64_t all_tiles = static_cast<int64_t>(tiles) * group;
    const int64_t share_low = all_tiles * piece / pieces, share_high = all_tiles * (piece + 1) / pieces;

    i32x4 k[TileT::kChunks], v[TileT::kChunks];
    {
        const T* const krow = a.k.at<T>(b, g) + j * a.k.n;
        const T* const vrow = a.v.at<T>(b, g) + j * a.v.n;
#pragma unroll
        for (int c = 0; c < TileT::kChunks; ++c) {
            const int d = (2 * c + half) * kPerFrag<T>;
            k[c] = v[c] = i32x4{0, 0, 0, 0};
            if (j < len) {
                k[c] = load_row<T, VEC>(krow, d, a.D);
                v[c] = load_row<T, VEC>(vrow, d, a.D);
            }
        }
    }
    f32x16 dk[kOut] = {}, dv[kOut] = {};
    float* const skew = skews + wave * kSkewFloats + 16;
    const bool biased = BIAS && (VEC || a.bias != nullptr);
    const float factor = biased ? 1.f : a.scale_log2;
    float* const mine = sums + wave * entries;
    if (summed)
        for (int i = threadIdx.x; i < kWaves * kSkewFloats; i += kThreads) skews[i] = 0.f;

    for (int hh = 0; hh < group; ++hh) {
        const int h = g * group + hh;
        const int from = t_first + static_cast<int>(max(share_low - static_cast<int64_t>(hh) * tiles, int64_t(0)));
        const int to = t_first + static_cast<int>(min(share_high - static_cast<int64_t>(hh) * tiles, int64_t(tiles)));
        float* const bucket_part =
            summed ? dbias_part + ((static_cast<int64_t>(b) * a.H + h) * (cut.units() + cut.first_units()) +
                                   (FIRST ? cut.units() : 0) + unit) * a.bk.count : nullptr;
        if (from >= to) {
            if (summed)
                for (int i = threadIdx.x; i < a.bk.count; i += kThreads) bucket_part[i] = 0.f;
            continue;
        }
        // Where all offsets are beyond the reach, one value serves all and one bucket takes all.
        const bool all_far = i_low + from * TQ + shift - (j0 + (FIRST ? 31 : kRows - 1)) >= a.reach;
        __syncthreads();
        if (biased) {
            if (!all_far) fill_bias<T>(a, h, table, edges);
            else if (threadIdx.x == 0)
                table[entries - 1] = bias_log2(to_float(static_cast<const T*>(a.bias)[static_cast<int64_t>(a.bk.n) * a.H + h]));
        }
        if (summed && !all_far)
            for (int i = threadIdx.x; i < kWaves * entries; i += kThreads) sums[i] = 0.f;
        float far_early = 0.f, far_late = 0.f;  // ds of offsets beyond the reach
        const T* const q = a.q.at<T>(b, h);
        const T* const go = grad.at<T>(b, h);
        const int64_t stats = (static_cast<int64_t>(b) * a.H + h) * a.Q;
        Stage<T, DP, TQ, VEC> qs, gs;
        float st = 0.f;
        int odd_rows = 0;  // lanes 0 .. TQ / 32: whether any of the 32 rows that the tile meets there is a coarse one
        const int groups_32 = (a.Q + 31) / 32;
        const auto flags = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<int*>(coarse_in + (static_cast<int64_t>(b) * a.H + h) * groups_32), 0, 4 * groups_32, kRawBuffer);
        auto fetch = [&](int t) {
            const int i0 = i_low + t * TQ;
            odd_rows = __builtin_amdgcn_raw_buffer_load_b32(flags, lane <= TQ / 32 ? 4u * (i0 / 32 + lane) : 0x80000000u, 0, 0);
            qs.load(q, a.q.n, i0, i_high, a.D);
            gs.load(go, grad.n, i0, i_high, a.D);
            if (threadIdx.x < 2 * TQ) {
                const bool is_lse = threadIdx.x < TQ;
                const int i = i0 + threadIdx.x % TQ;
                st = is_lse ? kInf : 0.f;
                if (i < i_high) st = (is_lse ? lse_in : delta_in)[stats + i];
            }
        };
        char* set = lds;
        // The shares of coarse rows (1 for others) are multiplied into their gradients and
        // delta, on which all of a row's sums depend linearly: as factors of the
        // weights they took 4 to 7 % more of the whole kernel.  16-bit gradients are
        // rounded once more thereby.
        auto put = [&](int t) {
            qs.store(set);
            if (ballot(odd_rows != 0) != 0) {
                auto share = [&](int row) {
                    const int i = i_low + t * TQ + row;
                    return i < i_high ? share_in[stats + i] : 1.f;
                };
                gs.scale(share);
                int thread = threadIdx.x;
                asm volatile("" : "+v"(thread));  // as in scale()
                if (thread >= TQ && thread < 2 * TQ) st *= share(thread - TQ);
            }
            gs.store(set + kTileBytes);
            if (threadIdx.x < 2 * TQ) reinterpret_cast<float*>(set + 2 * kTileBytes)[threadIdx.x] = st;
        };
        fetch(from);
        put(from);
        __syncthreads();
        for (int t = from; t < to; ++t) {
            if (t + 1 < to) fetch(t + 1);
            const char* const qtile = set;
            const char* const gtile = set + kTileBytes;
            const float* const stat = reinterpret_cast<const float*>(set + 2 * kTileBytes);
            const int p0 = i_low + t * TQ + shift;  // position of the tile's first row
            if (w_any && meets(p0)) {
                const bool whole = wholly(p0);
                const int near = p0 - w0;
                const bool far = near - 31 >= a.reach || near + TQ - 1 <= -a.reach;
#pragma unroll
                for (int u = 0; u < kSub; ++u) {
                    if (FIRST && (t * kSub + u) % kWaves != wave) continue;
                    const int own = 32 * (sub + u);  // first row of the piece
                    RowFrags<T, DP> qf, gf;
                    qf.load(qtile, own);
                    if (!kTight) gf.load(gtile, own);
                    f32x4 lse[4], delta[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        lse[e] = *reinterpret_cast<const f32x4*>(stat + own + 8 * e + 4 * half);
                        delta[e] = *reinterpret_cast<const f32x4*>(stat + TQ + own + 8 * e + 4 * half);
                    }
                    keep_order();
                    f32x16 s = qf.times(k);
                    if (kTight) gf.load(gtile, own);
                    const f32x16 dp = gf.times(v);
                    ColumnFrags<T, DP> qc[2], gc[2];  // of this chunk of queries and the next
                    gc[0].load(gtile, own);
                    qc[0].load(qtile, own);
                    keep_order();
                    if (biased) {
                        s *= a.scale_log2;
                        if (far) {
                            s += table[near > 0 ? entries - 1 : 0];
                        } else {
                            const float* const from = table + near - lane % 32 + 4 * half + own + a.reach + kMargin;
#pragma unroll
                            for (int r = 0; r < 16; ++r) s[r] += from[8 * (r / 4) + r % 4];
                        }
                    }
                    float w[16], ds[16];
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        w[r] = exp2_fast(__builtin_fmaf(s[r], factor, -lse[r / 4][r % 4]));
                        ds[r] = w[r] * (dp[r] - delta[r / 4][r % 4]);
                    }
                    if (!whole) {
                        const int p = p0 + own + 4 * half - see_low;
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if ((static_cast<uint32_t>(p + 8 * (r / 4) + r % 4) >= see_count) != other) w[r] = ds[r] = 0.f;
                    }
                    constexpr int kSteps = 16 / kPerFrag<T>;
#pragma unroll
                    for (int c = 0; c < kSteps; ++c) {
                        if (c + 1 < kSteps) {
                            gc[(c + 1) % 2].load(gtile, own + (c + 1) * TileT::kRowsPerFrag);
                            qc[(c + 1) % 2].load(qtile, own + (c + 1) * TileT::kRowsPerFrag);
                        }
                        keep_order();
                        gc[c % 2].add(as_fragment<T>(&w[c * kPerFrag<T>]), dv);
                        qc[c % 2].add(as_fragment<T>(&ds[c * kPerFrag<T>]), dk);
                    }
                    if (!summed) continue;
                    if (!FIRST && j >= len) {  // keys of zeros with scores of their own
#pragma unroll
                        for (int r = 0; r < 16; ++r) ds[r] = 0.f;
                    }
                    if (far) {
                        float all = 0.f;
#pragma unroll
                        for (int r = 0; r < 16; ++r) all += ds[r];
                        if (near > 0) far_early += all;
                        else far_late += all;
                    } else {
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            if (lane % 32 / 16 == x) {
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    *reinterpret_cast<f32x4*>(skew + lane % 16 * kSkewRow + 8 * e + 4 * half) =
                                        f32x4{ds[4 * e], ds[4 * e + 1], ds[4 * e + 2], ds[4 * e + 3]};
                            }
                            lanes_exchange();
                            float all[4] = {};
#pragma unroll
                            for (int r = 0; r < 16; ++r) all[r % 4] += skew[r * (kSkewRow + 1) + lane - 16];
                            mine[near + own - 16 * x + lane - 16 + a.reach + kMargin] += (all[0] + all[1]) + (all[2] + all[3]);
                            lanes_exchange();
                        }
                    }
                }
            }
            set = set == lds ? lds + kSet : lds;
            if (t + 1 < to) put(t + 1);
            __syncthreads();
        }
        if (summed) {
            far_early = wave_sum(far_early);
            far_late = wave_sum(far_late);
            if (all_far) {
                if (lane == 0) sums[wave] = far_early;
                __syncthreads();
                for (int i = threadIdx.x; i < a.bk.count; i += kThreads)
                    bucket_part[i] = i == a.bk.n ? (sums[0] + sums[1]) + (sums[2] + sums[3]) : 0.f;
                continue;
            }
            if (lane == 0) {
                mine[entries - 1] += far_early;
                mine[0] += far_late;
            }
            __syncthreads();
            for (int i = threadIdx.x; i < entries; i += kThreads) {
                float all = sums[i];
#pragma unroll
                for (int w = 1; w < kWaves; ++w) all += sums[w * entries + i];
                sums[i] = all;
            }
            __syncthreads();
            add_buckets(a.bk, edges, sums, entries, a.reach + kMargin, bucket_part);
        }
    }

    if constexpr (SPLIT == 2) {
        float* const other = reinterpret_cast<float*>(lds) + wave % 2 * 32 * kOut * kWave;
        __syncthreads();
        if (wave >= 2) {
            put_sums(other, dk);
            put_sums(other + 16 * kOut * kWave, dv);
        }
        __syncthreads();
        if (wave >= 2) return;
        get_sums(other, dk, 1.f, 1.f);
        get_sums(other + 16 * kOut * kWave, dv, 1.f, 1.f);
    }
    // Key `key` of the block, formed again.
    auto again = [&](int key, Needed need, CarefulPair<T>& ck, CarefulPair<T>& cv) {
        const bool d0 = lane < a.D, d1 = lane + kWave < a.D;
        need = {need.k0 && d0, need.k1 && d1, need.v0 && d0, need.v1 && d1};
        for (int hh = 0; hh < group; ++hh) {
            const int64_t before = static_cast<int64_t>(hh) * tiles;
            const int from = t_first + static_cast<int>(max(share_low - before, int64_t(0)));
            const int to = t_first + static_cast<int>(min(share_high - before, static_cast<int64_t>(tiles)));
            if (careful_key<T>(a, grad, lse_in, delta_in, share_in, b, g * group + hh, j0 + key, i_low + from * TQ,
                               min(i_low + to * TQ, i_high), FIRST, len, need, ck, cv))
                break;
        }
    };
    // Keys behind the cloud's length have no gradient.
    float odd = 0.f;  // NaN where anything is not finite
#pragma unroll
    for (int d = 0; d < kOut; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            dk[d][r] = j < len ? dk[d][r] * a.scale : 0.f;
            dv[d][r] = j < len ? dv[d][r] : 0.f;
            odd += dk[d][r] * 0.f + dv[d][r] * 0.f;
        }
    float* const parts = part + bg * cut.floats(DP);
    if constexpr (FIRST) {
        // The waves' sums, added in order; then the part: (unit, dk or dv, key, DP).
        constexpr int kRow = DP + 4;
        float* const all = reinterpret_cast<float*>(lds);
        for (int w = 0; w < kWaves; ++w) {
            __syncthreads();
            if (w != wave) continue;
#pragma unroll
            for (int d = 0; d < kOut; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    f32x4* const x = reinterpret_cast<f32x4*>(all + lane % 32 * kRow + 32 * d + 8 * e + 4 * half);
                    f32x4* const y = reinterpret_cast<f32x4*>(all + (32 + lane % 32) * kRow + 32 * d + 8 * e + 4 * half);
                    const f32x4 zero = {};
                    const f32x4 xk = {dk[d][4 * e], dk[d][4 * e + 1], dk[d][4 * e + 2], dk[d][4 * e + 3]};
                    const f32x4 xv = {dv[d][4 * e], dv[d][4 * e + 1], dv[d][4 * e + 2], dv[d][4 * e + 3]};
                    *x = (w == 0 ? zero : *x) + xk;
                    *y = (w == 0 ? zero : *y) + xv;
                }
        }
        __syncthreads();
        float* const dst = parts + static_cast<int64_t>(cut.kept()) * 2 * cut.rows * DP + static_cast<int64_t>(unit) * 2 * 32 * DP;
        auto get = [&](int which, int key, int d) { return d < DP ? all[(32 * which + key) * kRow + d] : 0.f; };
        auto set = [&](int which, int key, int d, float x) {
            if (d < DP) dst[(32 * which + key) * DP + d] = x;
        };
        uint32_t bad = 0;
        for (int key = wave; key < 32; key += kWaves) {
            const float k0 = get(0, key, lane), k1 = get(0, key, lane + kWave), v0 = get(1, key, lane), v1 = get(1, key, lane + kWave);
            set(0, key, lane, k0), set(0, key, lane + kWave, k1), set(1, key, lane, v0), set(1, key, lane + kWave, v1);
            if (ballot(!finite((k0 + k1) + (v0 + v1))) != 0) bad |= 1u << key;
        }
        if (bad == 0) return;
        __threadfence();  // what is written again comes behind these stores
        while (bad != 0) {
            const int key = __builtin_ctz(bad);
            bad &= bad - 1;
            const Needed need = {!finite(get(0, key, lane)), !finite(get(0, key, lane + kWave)), !finite(get(1, key, lane)),
                                 !finite(get(1, key, lane + kWave))};
            CarefulPair<T> ck, cv;
            if (j0 + key < exist) again(key, need, ck, cv);
            if (need.k0) set(0, key, lane, ck.x0);
            if (need.k1) set(0, key, lane + kWave, ck.x1);
            if (need.v0) set(1, key, lane, cv.x0);
            if (need.v1) set(1, key, lane + kWave, cv.x1);
        }
        return;
    }
    uint64_t bad = ballot(odd != 0.f);
    bad = (bad | bad >> 32) & 0xffffffffu;
    const bool parted = cut.parted(block);
    // (unit, dk or dv, key of the block, DP), or the results.
    float* const dst = parts + (static_cast<int64_t>(unit) * 2 * kRows + (j - j0)) * DP;
    const int64_t to = ((static_cast<int64_t>(b) * a.N + j) * a.G + g) * a.D;
    if (parted) {
#pragma unroll
        for (int d = 0; d < kOut; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                store4<float, true>(dst, 32 * d + 8 * e + 4 * half, DP, dk[d], 4 * e);
                store4<float, true>(dst + kRows * DP, 32 * d + 8 * e + 4 * half, DP, dv[d], 4 * e);
            }
    } else if (j < a.N) {
#pragma unroll
        for (int d = 0; d < kOut; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                store4<T, VEC>(dk_out + to, 32 * d + 8 * e + 4 * half, a.D, dk[d], 4 * e);
                store4<T, VEC>(dv_out + to, 32 * d + 8 * e + 4 * half, a.D, dv[d], 4 * e);
            }
    }
    if (bad == 0) return;
    const uint64_t odd_k = odd_values(dk), odd_v = odd_values(dv);
    __threadfence();  // what is written again comes behind the keys' stores
    while (bad != 0) {
        const int r = __builtin_ctzll(bad);
        bad &= bad - 1;
        const int key = w0 - j0 + r;
        const Needed need = {odd_value(odd_k, r, lane), odd_value(odd_k, r, lane + kWave), odd_value(odd_v, r, lane),
                             odd_value(odd_v, r, lane + kWave)};
        CarefulPair<T> ck, cv;
        again(key, need, ck, cv);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int d = lane + x * kWave;
            const float yk = x == 0 ? ck.x0 : ck.x1, yv = x == 0 ? cv.x0 : cv.x1;
            const bool nk = x == 0 ? need.k0 : need.k1, nv = x == 0 ? need.v0 : need.v1;
            if (parted && d < DP) {
                float* const at = parts + (static_cast<int64_t>(unit) * 2 * kRows + key) * DP + d;
                if (nk) at[0] = yk;
                if (nv) at[kRows * DP] = yv;
            } else if (!parted && d < a.D) {
                const int64_t at = ((static_cast<int64_t>(b) * a.N + j0 + key) * a.G + g) * a.D + d;
                if (nk) dk_out[at] = from_float<T>(yk);
                if (nv) dv_out[at] = from_float<T>(yv);
            }
        }
    }
}

// The parts' sums, in their order: a thread four values of a key.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_join_kernel(const Args a, const float* __restrict__ part, int DP,
                                                                  T* __restrict__ dk, T* __restrict__ dv,
                                                                  const Pieces cut) {
    const int blocks = cut.joined_blocks(), bg = blockIdx.x / blocks, block = blockIdx.x % blocks;
    const int b = bg / a.G, g = bg % a.G;
    const int64_t each = static_cast<int64_t>(2) * cut.rows * DP;
    const float* const parts = part + bg * cut.floats(DP);
    const int at = 4 * static_cast<int>(blockIdx.y * kThreads + threadIdx.x);  // of 2 x rows x DP
    const int which = at / (cut.rows * DP), key = at / DP % cut.rows, d = at % DP, j = block * cut.rows + key;
    if (which > 1 || d >= a.D || j >= a.N) return;
    // Eight parts are asked for at once: each comes from memory.
    f32x4 all = {};
    auto add = [&](const float* from, int64_t step, int count) {
        constexpr int kAtOnce = 8;
        for (int i = 0; i < count; i += kAtOnce) {
            f32x4 x[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) x[u] = *reinterpret_cast<const f32x4*>(from + min(i + u, count - 1) * step);
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
                if (i + u < count) all += x[u];
        }
    };
    add(parts + static_cast<int64_t>(block) * cut.of_rest * each + at, each, cut.of_rest);
    if (j / 32 < cut.groups)
        add(parts + cut.kept() * each + static_cast<int64_t>(j / 32) * cut.of_first * 2 * 32 * DP + (which * 32 + j % 32) * DP + d,
            2 * 32 * DP, cut.of_first);
    T* const dst = (which == 0 ? dk : dv) + ((static_cast<int64_t>(b) * a.N + j) * a.G + g) * a.D;
#pragma unroll
    for (int f = 0; f < 4; ++f)
        if (d + f < a.D) dst[d + f] = from_float<T>(all[f]);
}

// Blocks of 64 keys where those of 128 are few, and pieces where these are: up
// to two blocks a compute unit (512; a few more would be a round of their own),
// of 4 tiles or more.
Pieces pieces_of(const Args& a, int inner, bool may_split) {
    Pieces cut{kOuter, (a.N + kOuter - 1) / kOuter, 1, 0, 1};
    const int64_t heads = static_cast<int64_t>(a.B) * a.G;
    if (heads == 0 || a.N == 0 || a.H == 0 || a.Q == 0) return cut;
    if (may_split && few_blocks(cut.key_blocks * heads)) {
        cut.rows = kOuter / 2;
        cut.key_blocks = (a.N + cut.rows - 1) / cut.rows;
        inner = Cut<float, 2>::kInnerRows;
    }
    auto pieces = [&](int64_t rows, int64_t blocks, int64_t least) {
        const int64_t tiles = (rows + inner - 1) / inner * (a.H / a.G);
        return static_cast<int>(std::max<int64_t>(1, std::min(512 / blocks, tiles / least)));
    };
    cut.of_rest = pieces(std::min<int64_t>(a.Q, static_cast<int64_t>(a.causal ? 1 : 2) * a.window + cut.rows),
                         cut.key_blocks * heads, 4);
    if (a.sinks > 0 && a.window < a.N) {
        cut.groups = (a.sinks + 31) / 32;
        cut.of_first = std::min(32, pieces(a.Q, cut.groups * heads, 2));
    }
    return cut;
}

int padded(int64_t D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }

struct Workspace {
    Pieces cut;
    size_t delta, share, coarse, bias, part, bytes;
};

Workspace workspace_of(const Args& a, int type, bool may_split) {
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t rows = static_cast<size_t>(a.B) * a.H;
    Workspace w{};
    w.cut = pieces_of(a, type == POINTOPS_F32 ? kInner<float> : kInner<f16>, may_split);
    const size_t units = static_cast<size_t>(w.cut.units()) + w.cut.first_units();
    w.delta = 0;
    w.share = up(rows * a.Q * sizeof(float));
    w.coarse = 2 * w.share;
    w.bias = w.coarse + up(rows * ((a.Q + 31) / 32) * sizeof(int));
    w.part = w.bias + (a.bias != nullptr ? up(rows * units * a.bk.count * sizeof(float)) : 0);
    w.bytes = w.part + static_cast<size_t>(a.B) * a.G * w.cut.floats(padded(a.D)) * sizeof(float);
    return w;
}

struct Grads {
    const void* out;
    const float* lse;
    Rows grad;
    void *dq, *dk, *dv, *dbias;
    char* workspace;
};

template <typename T>
constexpr int kType = sizeof(T) == 4 ? POINTOPS_F32 : __is_same(T, f16) ? POINTOPS_F16 : POINTOPS_BF16;

template <typename T, int DP, bool VEC, bool BIAS>
hipError_t launch_backward(const Args& a, const Grads& x, hipStream_t stream) {
    using TileT = Tile<T, DP>;
    constexpr bool kSplit = VEC && kSplits<T, DP>;
    const Workspace w = workspace_of(a, kType<T>, kSplit);
    const Pieces cut = w.cut;
    float* const delta = reinterpret_cast<float*>(x.workspace + w.delta);
    float* const share = reinterpret_cast<float*>(x.workspace + w.share);
    int* const coarse = reinterpret_cast<int*>(x.workspace + w.coarse);
    float* const dbias_part = x.dbias != nullptr ? reinterpret_cast<float*>(x.workspace + w.bias) : nullptr;
    float* const part = reinterpret_cast<float*>(x.workspace + w.part);
    const int64_t heads = static_cast<int64_t>(a.B) * a.G, grid_k = cut.units() * heads, grid_first = cut.first_units() * heads;
    const bool split_q = kSplit && few_blocks((static_cast<int64_t>(a.Q) + kOuter - 1) / kOuter * a.B * a.H);
    const bool split_k = kSplit && cut.rows < kOuter;
    const int64_t rows_q = split_q ? kOuter / 2 : kOuter;
    const int64_t grid_q = (static_cast<int64_t>(a.Q) + rows_q - 1) / rows_q * a.B * a.H;
    if (grid_q > INT32_MAX || grid_k > INT32_MAX || grid_first > INT32_MAX) return hipErrorInvalidValue;

    auto tiles = [](bool split) { return 4 * (split ? Cut<T, 2>::kInnerRows : kInner<T>) * static_cast<size_t>(TileT::kStride); };
    const size_t entries = bias_entries(a.reach), table = a.bias != nullptr ? 4 * (entries + a.bk.n) : 0;
    if (grid_q > 0) {
        auto* kernel = attention_grad_query_kernel<T, DP, VEC, BIAS, 1>;
        if constexpr (kSplit)
            if (split_q) kernel = attention_grad_query_kernel<T, DP, VEC, BIAS, 2>;
        const size_t lds = tiles(split_q) + table;
        if (lds > kLdsFree) {
            static std::atomic<uint64_t> allowed[2];
            const hipError_t err = allow_lds(kernel, allowed[split_q], tiles(split_q) + 4 * (bias_entries(kMaxReach) + 255));
            if (err != hipSuccess) return err;
        }
        hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(grid_q)), dim3(kThreads), lds, stream, a,
                           static_cast<const T*>(x.out), x.lse, x.grad, delta, share, coarse, static_cast<T*>(x.dq), a.bias != nullptr);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    if (grid_k > 0) {
        // The tiles, their rows' statistics, the bias's table; with its sums also the skews and the waves' sums.
        auto lds_for = [&](bool split, size_t n, size_t edges, bool sums) {
            return tiles(split) + tiles(split) / TileT::kStride * 4 + 4 * ((n + 3) / 4 * 4 + edges) +
                   (sums ? 4 * kWaves * (kSkewFloats + n) : 0);
        };
        auto launch = [&](auto* kernel, bool split, int64_t grid, std::atomic<uint64_t>& allowed) {
            const size_t lds = a.bias != nullptr ? lds_for(split, entries, a.bk.n, dbias_part != nullptr)
                                                 : lds_for(split, 0, 0, false);
            if (lds > kLdsFree) {
                const hipError_t err = allow_lds(kernel, allowed, lds_for(split, bias_entries(kMaxReach), 255, true));
                if (err != hipSuccess) return err;
            }
            hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(grid)), dim3(kThreads), lds, stream, a, x.lse, delta, share, coarse, x.grad,
                               static_cast<T*>(x.dk), static_cast<T*>(x.dv), part, dbias_part, cut);
            return hipGetLastError();
        };
        static std::atomic<uint64_t> allowed[3];
        hipError_t err = hipSuccess;
        if constexpr (kSplit)
            if (split_k) err = launch(attention_grad_key_kernel<T, DP, VEC, BIAS, false, 2>, true, grid_k, allowed[0]);
        if (!split_k) err = launch(attention_grad_key_kernel<T, DP, VEC, BIAS, false, 1>, false, grid_k, allowed[1]);
        if (err == hipSuccess && grid_first > 0)
            err = launch(attention_grad_key_kernel<T, DP, VEC, BIAS, true, 1>, false, grid_first, allowed[2]);
        if (err != hipSuccess) return err;
        if (cut.kept() > 0) {
            const dim3 grid(static_cast<uint32_t>(heads * cut.joined_blocks()), 2 * cut.rows * DP / (4 * kThreads));
            hipLaunchKernelGGL(attention_join_kernel<T>, grid, dim3(kThreads), 0, stream, a, part, DP,
                               static_cast<T*>(x.dk), static_cast<T*>(x.dv), cut);
            err = hipGetLastError();
            if (err != hipSuccess) return err;
        }
    }
    if (x.dbias == nullptr || a.H == 0) return hipSuccess;
    return join_buckets(dbias_part, a.B, a.H, cut.units() + cut.first_units(), a.bk.count, kType<T>, a.bias, x.dbias, stream);
}

template <typename T>
hipError_t backward(const Args& a, const Grads& x, hipStream_t stream) {
    const bool vec = vector_rows<T>(a.q, a.D) && vector_rows<T>(a.k, a.D) && vector_rows<T>(a.v, a.D) &&
                     vector_rows<T>(x.grad, a.D) && reinterpret_cast<uintptr_t>(x.out) % 16 == 0;
    return with_width(a.D, [&](auto width) {
        constexpr int DP = decltype(width)::value;
        if (!vec) return launch_backward<T, DP, false, true>(a, x, stream);
        return a.bias != nullptr ? launch_backward<T, DP, true, true>(a, x, stream) : launch_backward<T, DP, true, false>(a, x, stream);
    });
}

}  // namespace
}  // namespace attn
}  // namespace pointops

extern "C" {

size_t pointops_attention_backward_workspace_bytes(const pointops_attention* in) {
    using namespace pointops::attn;
    Args a;
    if (!read_args(in, &a)) return 0;
    // Whether rows are read in 16-byte pieces depends on the gradient's strides too.
    return std::max(workspace_of(a, in->type, true).bytes, workspace_of(a, in->type, false).bytes);
}

hipError_t pointops_attention_backward(const pointops_attention* in, const void* out, const float* lse,
                                       const void* grad_out, const int64_t* grad_stride, void* dq, void* dk, void* dv,
                                       void* dbias, void* workspace, hipStream_t stream) {
    using namespace pointops::attn;
    Args a;
    if (!read_args(in, &a)) return hipErrorInvalidValue;
    if (dbias != nullptr && a.bias == nullptr) return hipErrorInvalidValue;
    // (Of sides that are empty the others' gradients are zeros, written as any.)
    const bool queries = a.B > 0 && a.H > 0 && a.Q > 0, keys = a.B > 0 && a.G > 0 && a.N > 0;
    if (queries && (in->q == nullptr || out == nullptr || lse == nullptr || grad_out == nullptr || grad_stride == nullptr ||
                    dq == nullptr))
        return hipErrorInvalidValue;
    if (keys && (in->k == nullptr || in->v == nullptr || dk == nullptr || dv == nullptr)) return hipErrorInvalidValue;
    if ((queries || keys) && workspace == nullptr && pointops_attention_backward_workspace_bytes(in) != 0) return hipErrorInvalidValue;
    Grads x{out, lse, {}, dq, dk, dv, dbias, static_cast<char*>(workspace)};
    if (grad_stride != nullptr) x.grad = {grad_out, grad_stride[0], grad_stride[1], grad_stride[2]};
    switch (in->type) {
        case POINTOPS_F32: return backward<float>(a, x, stream);
        case POINTOPS_F16: return backward<f16>(a, x, stream);
        default: return backward<bf16>(a, x, stream);
    }
}

}  // extern "C"
