// Attention within a window of the order: the backward pass.
//
//   dv_j = sum_i p_ij do_i            ds_ij = p_ij (do_i v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j      dk_j = scale sum_i ds_ij q_i
//   delta_i = do_i o_i                dbias[bucket] = sum of ds_ij with i - j in the bucket
//
// The weights are formed again from the scores and the forward's logarithms of
// the sums.  Two kernels, so that every sum has one owner and a fixed order
// (no atomics: results do not change from run to run): one holds 128 queries
// in registers and passes over their keys (delta, dq and the bias's sums by
// offset), the other holds 128 keys and passes over the queries that see them,
// all heads that share the key head in turn (dk, dv).  The first keys that
// every query sees are read by all rows: their pass is cut into pieces whose
// 32-bit sums a last kernel joins.  ds and p are rounded to the inputs' type
// for the second products, as the forward's weights are.
#include <algorithm>
#include <atomic>

#include "attention.hpp"

namespace pointops {
namespace attn {
namespace {

// Sums of ds by offset: one table a wave and half-wave (no two lanes of an
// addition share an entry, and one wave's additions keep their order).
constexpr int kSums = 2 * kWaves;

template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(kThreads, (sizeof(T) == 4 && DP > 64) ? 1 : 2) void attention_grad_query_kernel(
    const Args a, const T* __restrict__ out, const float* __restrict__ lse_in, const Rows grad,
    float* __restrict__ delta_out, T* __restrict__ dq_out, float* __restrict__ dbias_part) {
    using TileT = Tile<T, DP>;
    constexpr int TK = kInner<T>, kOut = DP / 32;
    extern __shared__ char lds[];
    char* const ktile = lds;
    char* const vtile = lds + TK * TileT::kStride;
    float* const table = reinterpret_cast<float*>(lds + 2 * TK * TileT::kStride);
    const int entries = bias_entries(a.reach);

    const int lane = lane_id(), half = lane / 32, wave = uniform(threadIdx.x / kWave);
    const uint32_t blocks = (a.Q + kOuter - 1) / kOuter;
    const uint32_t blk = xcd_local_block(blockIdx.x, gridDim.x);
    const int bh = static_cast<int>(blk / blocks), b = bh / a.H, h = bh % a.H, g = h / (a.H / a.G);
    const int iblock = static_cast<int>(blocks - 1 - blk % blocks), i0 = iblock * kOuter;
    const int len = a.length(b), shift = a.N - a.Q;
    const bool biased = a.bias != nullptr, summed = dbias_part != nullptr;
    float* const sums = table + entries;  // kSums tables of `entries`, behind them the edges
    if (biased) {
        fill_bias<T>(a, h, table, reinterpret_cast<int*>(sums + (summed ? kSums * entries : 0)));
        if (summed)
            for (int i = threadIdx.x; i < kSums * entries; i += kThreads) sums[i] = 0.f;
    }

    const int rows = min(kOuter, a.Q - i0);
    const int p_first = max(i0 + shift, 0), p_last = min(i0 + shift + rows, len) - 1;
    int t = 0, t_first_end = 0, t_low = 0, t_high = -1;
    if (p_first <= p_last) {
        t_first_end = (seen_first(a, p_last, len) + TK - 1) / TK;
        t_low = max(t_first_end, seen_low(a, p_first) / TK);
        t_high = seen_high(a, p_last, len) / TK;
        t = t_first_end > 0 ? 0 : t_low;
    }
    const int t_end = max(t_first_end, t_high + 1);

    const int w0 = i0 + 32 * wave + shift;
    const int w_count = min(32, i0 + rows - (i0 + 32 * wave));
    const int w_first = max(w0, 0), w_last = min(w0 + w_count, len) - 1;
    const bool w_any = w_first <= w_last, w_whole = w_any && w0 >= 0 && w0 + w_count <= len;
    const int row = i0 + 32 * wave + lane % 32, p = row + shift;
    const bool exists = row < a.Q && p >= 0 && p < len;
    const Seen seen = seen_by(a, p, len);

    i32x4 q[TileT::kChunks], go[TileT::kChunks];
    float delta = 0.f, lse = kInf;
    {
        const T* const qrow = a.q.at<T>(b, h) + row * a.q.n;
        const T* const grow = grad.at<T>(b, h) + row * grad.n;
        const int64_t at = (static_cast<int64_t>(b) * a.Q + row) * a.H + h;
        const T* const orow = out + at * a.D;
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
        const int64_t stat = (static_cast<int64_t>(b) * a.H + h) * a.Q + row;
        if (exists) lse = lse_in[stat];
        if (row < a.Q && half == 0) delta_out[stat] = delta;
    }
    const T* const k = a.k.at<T>(b, g);
    const T* const v = a.v.at<T>(b, g);
    f32x16 dq[kOut] = {};
    float far_early = 0.f, far_late = 0.f;  // ds of offsets beyond the reach

    Stage<T, DP, TK, VEC> ks, vs;
    if (t < t_end) {
        ks.load(k, a.k.n, t * TK, 0, len, a.D);
        vs.load(v, a.v.n, t * TK, 0, len, a.D);
    }
    while (t < t_end) {
        __syncthreads();
        ks.store(ktile);
        vs.store(vtile);
        __syncthreads();
        const int j0 = t * TK;
        ++t;
        if (t >= t_first_end && t < t_low) t = t_low;
        if (t < t_end) {
            ks.load(k, a.k.n, t * TK, 0, len, a.D);
            vs.load(v, a.v.n, t * TK, 0, len, a.D);
        }
        if (!w_any) continue;
        const bool meets = (j0 <= seen_high(a, w_last, len) && j0 + TK > seen_low(a, w_first)) ||
                           j0 < seen_first(a, w_last, len);
        if (!meets) continue;
        const bool whole = w_whole && ((j0 + TK - 1 <= seen_high(a, w_first, len) && j0 >= seen_low(a, w_last)) ||
                                       j0 + TK <= seen_first(a, w_first, len));
        const int near = w0 - j0;
        const bool far = near - (TK - 1) >= a.reach || near + 31 <= -a.reach;
#pragma unroll
        for (int u = 0; u < TK / 32; ++u) {
            f32x16 s = {}, dp = {};
#pragma unroll
            for (int c = 0; c < TileT::kChunks; ++c) s = mma<T>(TileT::rows(ktile, 32 * u, c), q[c], s);
#pragma unroll
            for (int c = 0; c < TileT::kChunks; ++c) dp = mma<T>(TileT::rows(vtile, 32 * u, c), go[c], dp);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] *= a.scale_log2;
            const int at = near + lane % 32 - 4 * half - 32 * u + a.reach + kMargin;
            if (biased) {
                if (far) {
                    const float add = table[near > 0 ? entries - 1 : 0];
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] += add;
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] += table[at - (8 * (r / 4) + r % 4)];
                }
            }
            if (!whole) {
                const int j = j0 + 32 * u + 4 * half;
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!seen(j + 8 * (r / 4) + r % 4)) s[r] = -kInf;
            }
            float ds[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float w = exp2_fast(s[r] - lse);
                ds[r] = w * (dp[r] - delta);
                if (!whole && w == 0.f) ds[r] = 0.f;  // a masked key's infinity or NaN stays out
            }
            if (summed) {
                if (far) {
                    float all = 0.f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) all += ds[r];
                    if (near > 0) far_early += all;
                    else far_late += all;
                } else {
                    float* const mine = sums + (2 * wave + half) * entries + at;
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        __hip_atomic_fetch_add(mine - (8 * (r / 4) + r % 4), ds[r], __ATOMIC_RELAXED,
                                               __HIP_MEMORY_SCOPE_WORKGROUP);
                }
            }
#pragma unroll
            for (int c = 0; c < 16 / kPerFrag<T>; ++c) {
                const i32x4 w = as_fragment<T>(&ds[c * kPerFrag<T>]);
#pragma unroll
                for (int d = 0; d < kOut; ++d)
                    dq[d] = mma<T>(TileT::columns(ktile, 32 * u + c * TileT::kRowsPerFrag, 32 * d), w, dq[d]);
            }
        }
    }

    if (row < a.Q) {
        T* const dst = dq_out + ((static_cast<int64_t>(b) * a.Q + row) * a.H + h) * a.D;
#pragma unroll
        for (int d = 0; d < kOut; ++d) {
            dq[d] *= a.scale;
#pragma unroll
            for (int e = 0; e < 4; ++e) store4<T, VEC>(dst, 32 * d + 8 * e + 4 * half, a.D, dq[d], 4 * e);
        }
    }
    if (summed) {
        __syncthreads();
        far_early = wave_sum(far_early);
        far_late = wave_sum(far_late);
        if (lane == 0) {
            float* const mine = sums + 2 * wave * entries;
            mine[entries - 1] += far_early;
            mine[0] += far_late;
        }
        __syncthreads();
        float* const dst = dbias_part + (static_cast<int64_t>(bh) * blocks + iblock) * entries;
        for (int i = threadIdx.x; i < entries; i += kThreads) {
            float all = 0.f;
#pragma unroll
            for (int w = 0; w < kSums; ++w) all += sums[w * entries + i];
            dst[i] = all;
        }
    }
}

// A key block's share of the queries: pieces of the blocks that hold the first
// keys, which all later rows see, and the whole range of the others.
struct Pieces {
    int first_blocks;  // key blocks that are cut
    int pieces;        // into so many
};

template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(kThreads, 1) void attention_grad_key_kernel(
    const Args a, const float* __restrict__ lse_in, const float* __restrict__ delta_in, const Rows grad,
    T* __restrict__ dk_out, T* __restrict__ dv_out, float* __restrict__ part, const Pieces cut) {
    using TileT = Tile<T, DP>;
    constexpr int TQ = kInner<T>, kOut = DP / 32;
    extern __shared__ char lds[];
    char* const qtile = lds;
    char* const gtile = lds + TQ * TileT::kStride;
    float* const stat = reinterpret_cast<float*>(lds + 2 * TQ * TileT::kStride);  // lse, then delta
    float* const table = stat + 2 * TQ;
    const int entries = bias_entries(a.reach);

    const int lane = lane_id(), half = lane / 32, wave = uniform(threadIdx.x / kWave);
    const int key_blocks = (a.N + kOuter - 1) / kOuter;
    const uint32_t blocks = key_blocks + cut.first_blocks * (cut.pieces - 1);
    const uint32_t blk = xcd_local_block(blockIdx.x, gridDim.x);
    const int bg = static_cast<int>(blk / blocks), b = bg / a.G, g = bg % a.G;
    const int index = static_cast<int>(blk % blocks);
    const bool pieced = index < cut.first_blocks * cut.pieces;
    const int piece = pieced ? index % cut.pieces : 0;
    const int jblock = pieced ? index / cut.pieces : index - cut.first_blocks * (cut.pieces - 1);
    const int j0 = jblock * kOuter, len = a.length(b), shift = a.N - a.Q;
    const bool biased = a.bias != nullptr;
    const int group = a.H / a.G;

    // Queries that see any of the block's keys, by row.
    const int j_last = min(j0 + kOuter, len) - 1;
    int i_first = 0, i_last = -1;
    if (j_last >= j0) {
        const bool first = j0 < a.sinks;
        int p_low = a.causal ? j0 : first ? 0 : j0 - a.window + 1;
        int p_high = first || j_last > len - a.window ? len - 1 : j_last + a.window - 1;
        p_low = max(p_low, 0);
        p_high = min(p_high, len - 1);
        i_first = max(p_low - shift, 0);
        i_last = min(p_high - shift, a.Q - 1);
    }
    int t_first = i_first / TQ, t_end = i_last < i_first ? t_first : i_last / TQ + 1;
    if (pieced) {
        const int each = (t_end - t_first + cut.pieces - 1) / cut.pieces;
        t_first = min(t_first + piece * each, t_end);
        t_end = min(t_first + each, t_end);
    }
    const int i_low = max(-shift, 0), i_high = min(a.Q, len - shift);  // rows that exist

    // This wave's keys: one a lane column.
    const int w0 = j0 + 32 * wave;
    const int w_last = min(w0 + 32, len) - 1;
    const bool w_any = w0 <= w_last;
    const int j = w0 + lane % 32;
    // The lane's key is seen from positions low .. low + count - 1.
    const bool first_key = j < a.sinks;
    const int see_low = a.causal ? j : first_key ? 0 : j - a.window + 1;
    const int see_high = first_key || j > len - a.window ? len - 1 : j + a.window - 1;
    const uint32_t see_count = static_cast<uint32_t>(max(see_high - see_low + 1, 0));

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

    for (int hh = 0; hh < group; ++hh) {
        const int h = g * group + hh;
        __syncthreads();
        if (biased) fill_bias<T>(a, h, table, reinterpret_cast<int*>(table + entries));
        const T* const q = a.q.at<T>(b, h);
        const T* const go = grad.at<T>(b, h);
        const int64_t stats = (static_cast<int64_t>(b) * a.H + h) * a.Q;
        Stage<T, DP, TQ, VEC> qs, gs;
        float st = 0.f;
        auto fetch = [&](int t) {
            qs.load(q, a.q.n, t * TQ, i_low, i_high, a.D);
            gs.load(go, grad.n, t * TQ, i_low, i_high, a.D);
            if (threadIdx.x < 2 * TQ) {
                const bool is_lse = threadIdx.x < TQ;
                const int i = t * TQ + threadIdx.x % TQ;
                const bool there = i >= i_low && i < i_high;
                st = is_lse ? kInf : 0.f;
                if (there) st = (is_lse ? lse_in : delta_in)[stats + i];
            }
        };
        if (t_first < t_end) fetch(t_first);
        for (int t = t_first; t < t_end; ++t) {
            __syncthreads();
            qs.store(qtile);
            gs.store(gtile);
            if (threadIdx.x < 2 * TQ) stat[threadIdx.x] = st;
            __syncthreads();
            if (t + 1 < t_end) fetch(t + 1);
            if (!w_any) continue;
            const int p0 = t * TQ + shift;  // position of the tile's first row
            // Positions that all, or any, of the wave's keys are seen from.
            const int all_low = a.causal ? w_last : w_last < a.sinks ? 0 : w_last - a.window + 1;
            const int all_high = w_last < a.sinks ? len - 1 : w0 > len - a.window ? len - 1 : w0 + a.window - 1;
            const int any_low = a.causal ? w0 : w0 < a.sinks ? 0 : w0 - a.window + 1;
            const int any_high = w0 < a.sinks || w_last > len - a.window ? len - 1 : w_last + a.window - 1;
            if (p0 > any_high || p0 + TQ <= any_low) continue;
            const bool whole = p0 >= all_low && p0 + TQ - 1 <= all_high;
            const int near = p0 - w0;
            const bool far = near - 31 >= a.reach || near + TQ - 1 <= -a.reach;
#pragma unroll
            for (int u = 0; u < TQ / 32; ++u) {
                f32x16 s = {}, dp = {};
#pragma unroll
                for (int c = 0; c < TileT::kChunks; ++c) s = mma<T>(TileT::rows(qtile, 32 * u, c), k[c], s);
#pragma unroll
                for (int c = 0; c < TileT::kChunks; ++c) dp = mma<T>(TileT::rows(gtile, 32 * u, c), v[c], dp);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] *= a.scale_log2;
                if (biased) {
                    if (far) {
                        const float add = table[near > 0 ? entries - 1 : 0];
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[r] += add;
                    } else {
                        const float* const at = table + near - lane % 32 + 4 * half + 32 * u + a.reach + kMargin;
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[r] += at[8 * (r / 4) + r % 4];
                    }
                }
                if (!whole) {
                    const int p = p0 + 32 * u + 4 * half - see_low;
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (static_cast<uint32_t>(p + 8 * (r / 4) + r % 4) >= see_count) s[r] = -kInf;
                }
                float w[16], ds[16];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f32x4 lse = *reinterpret_cast<const f32x4*>(stat + 32 * u + 8 * e + 4 * half);
                    const f32x4 delta = *reinterpret_cast<const f32x4*>(stat + TQ + 32 * u + 8 * e + 4 * half);
#pragma unroll
                    for (int f = 0; f < 4; ++f) {
                        const int r = 4 * e + f;
                        w[r] = exp2_fast(s[r] - lse[f]);
                        ds[r] = w[r] * (dp[r] - delta[f]);
                        if (!whole && w[r] == 0.f) ds[r] = 0.f;
                    }
                }
#pragma unroll
                for (int c = 0; c < 16 / kPerFrag<T>; ++c) {
                    const i32x4 x = as_fragment<T>(&w[c * kPerFrag<T>]), y = as_fragment<T>(&ds[c * kPerFrag<T>]);
#pragma unroll
                    for (int d = 0; d < kOut; ++d) {
                        dv[d] = mma<T>(TileT::columns(gtile, 32 * u + c * TileT::kRowsPerFrag, 32 * d), x, dv[d]);
                        dk[d] = mma<T>(TileT::columns(qtile, 32 * u + c * TileT::kRowsPerFrag, 32 * d), y, dk[d]);
                    }
                }
            }
        }
    }

    // Keys behind the cloud's length were zeros with scores of their own: they
    // have no gradient.
    const float there = j < len ? 1.f : 0.f;
#pragma unroll
    for (int d = 0; d < kOut; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            dk[d][r] = there != 0.f ? dk[d][r] * a.scale : 0.f;
            dv[d][r] = there != 0.f ? dv[d][r] : 0.f;
        }
    if (pieced) {
        // (b g, first block, piece, dk or dv, key of the block, D)
        float* const dst = part + (((static_cast<int64_t>(bg) * cut.first_blocks + jblock) * cut.pieces + piece) * 2 * kOuter +
                                   (j - j0)) * DP;
#pragma unroll
        for (int d = 0; d < kOut; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                store4<float, true>(dst, 32 * d + 8 * e + 4 * half, DP, dk[d], 4 * e);
                store4<float, true>(dst + kOuter * DP, 32 * d + 8 * e + 4 * half, DP, dv[d], 4 * e);
            }
    } else if (j < a.N) {
        const int64_t at = ((static_cast<int64_t>(b) * a.N + j) * a.G + g) * a.D;
#pragma unroll
        for (int d = 0; d < kOut; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                store4<T, VEC>(dk_out + at, 32 * d + 8 * e + 4 * half, a.D, dk[d], 4 * e);
                store4<T, VEC>(dv_out + at, 32 * d + 8 * e + 4 * half, a.D, dv[d], 4 * e);
            }
    }
}

// The pieces' sums, in their order: one thread an element.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_join_kernel(const Args a, const float* __restrict__ part, int DP,
                                                                  T* __restrict__ dk, T* __restrict__ dv,
                                                                  const Pieces cut) {
    const int block = blockIdx.x, bg = block / cut.first_blocks, jblock = block % cut.first_blocks;
    const int b = bg / a.G, g = bg % a.G;
    const float* const src = part + static_cast<int64_t>(block) * cut.pieces * 2 * kOuter * DP;
    const int at = blockIdx.y * kThreads + threadIdx.x;  // of 2 x kOuter x DP
    const int which = at / (kOuter * DP), key = at / DP % kOuter, d = at % DP, j = jblock * kOuter + key;
    if (which > 1 || d >= a.D || j >= a.N) return;
    float all = 0.f;
    for (int i = 0; i < cut.pieces; ++i) all += src[static_cast<int64_t>(i) * 2 * kOuter * DP + at];
    (which == 0 ? dk : dv)[((static_cast<int64_t>(b) * a.N + j) * a.G + g) * a.D + d] = from_float<T>(all);
}

// The first keys' blocks take all later rows, the others window + 128 of them
// (two windows where later keys are seen too): pieces of about that length.
Pieces pieces_of(const Args& a) {
    if (a.sinks == 0 || a.N == 0) return {0, 1};
    const int64_t rows = static_cast<int64_t>(a.causal ? 1 : 2) * a.window + kOuter;
    const int64_t pieces = std::min<int64_t>(64, a.Q / std::max<int64_t>(rows, 512));
    if (pieces < 2) return {0, 1};
    return {(a.sinks + kOuter - 1) / kOuter, static_cast<int>(pieces)};
}

int padded(int64_t D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }

struct Workspace {
    size_t delta, bias, part, bytes;
};

Workspace workspace_of(const Args& a) {
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t rows = static_cast<size_t>(a.B) * a.H, blocks = (static_cast<size_t>(a.Q) + kOuter - 1) / kOuter;
    const Pieces cut = pieces_of(a);
    Workspace w{};
    w.delta = 0;
    w.bias = up(rows * a.Q * sizeof(float));
    w.part = w.bias + (a.bias != nullptr ? up(rows * blocks * bias_entries(a.reach) * sizeof(float)) : 0);
    w.bytes = w.part + (cut.pieces > 1 ? static_cast<size_t>(a.B) * a.G * cut.first_blocks * cut.pieces * 2 * kOuter *
                                             padded(a.D) * sizeof(float)
                                       : 0);
    return w;
}

// Allows a kernel the LDS that its largest bias tables need, once per device
// (the limit belongs to the process).
template <typename K>
hipError_t allow_lds(K kernel, std::atomic<uint64_t>& allowed, size_t most) {
    int dev = 0;
    const hipError_t err = hipGetDevice(&dev);
    if (err != hipSuccess) return err;
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if ((allowed.load(std::memory_order_acquire) & bit) != 0) return hipSuccess;
    const hipError_t set = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most));
    if (set == hipSuccess) allowed.fetch_or(bit, std::memory_order_release);
    return set;
}

constexpr size_t kLdsFree = 64 * 1024;  // what a launch may take without asking

struct Grads {
    const void* out;
    const float* lse;
    Rows grad;
    void *dq, *dk, *dv, *dbias;
    char* workspace;
};

template <typename T, int DP, bool VEC>
hipError_t launch_backward(const Args& a, const Grads& x, hipStream_t stream) {
    using TileT = Tile<T, DP>;
    const Workspace w = workspace_of(a);
    float* const delta = reinterpret_cast<float*>(x.workspace + w.delta);
    float* const dbias_part = x.dbias != nullptr ? reinterpret_cast<float*>(x.workspace + w.bias) : nullptr;
    float* const part = reinterpret_cast<float*>(x.workspace + w.part);
    const int64_t query_blocks = (static_cast<int64_t>(a.Q) + kOuter - 1) / kOuter;
    const int64_t key_blocks = (static_cast<int64_t>(a.N) + kOuter - 1) / kOuter;
    const Pieces cut = pieces_of(a);
    const int64_t grid_q = query_blocks * a.B * a.H;
    const int64_t grid_k = (key_blocks + static_cast<int64_t>(cut.first_blocks) * (cut.pieces - 1)) * a.B * a.G;
    if (grid_q > INT32_MAX || grid_k > INT32_MAX) return hipErrorInvalidValue;

    constexpr size_t tiles = 2 * kInner<T> * TileT::kStride;
    const size_t entries = bias_entries(a.reach);
    size_t lds = tiles;
    if (a.bias != nullptr) lds += 4 * (entries * (x.dbias != nullptr ? 1 + kSums : 1) + a.bk.n);
    auto* const by_query = attention_grad_query_kernel<T, DP, VEC>;
    if (lds > kLdsFree) {
        static std::atomic<uint64_t> allowed{0};
        const hipError_t err = allow_lds(by_query, allowed, tiles + 4 * ((1 + kSums) * bias_entries(kMaxReach) + 255));
        if (err != hipSuccess) return err;
    }
    if (grid_q > 0) {
        hipLaunchKernelGGL(by_query, dim3(static_cast<uint32_t>(grid_q)), dim3(kThreads), lds, stream, a,
                           static_cast<const T*>(x.out), x.lse, x.grad, delta, static_cast<T*>(x.dq), dbias_part);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    if (grid_k > 0) {
        lds = tiles + 8 * kInner<T> + (a.bias != nullptr ? 4 * (entries + a.bk.n) : 0);
        hipLaunchKernelGGL((attention_grad_key_kernel<T, DP, VEC>), dim3(static_cast<uint32_t>(grid_k)), dim3(kThreads),
                           lds, stream, a, x.lse, delta, x.grad, static_cast<T*>(x.dk), static_cast<T*>(x.dv), part, cut);
        hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
        if (cut.pieces > 1) {
            const dim3 grid(static_cast<uint32_t>(static_cast<int64_t>(a.B) * a.G * cut.first_blocks),
                            2 * kOuter * DP / kThreads);
            hipLaunchKernelGGL(attention_join_kernel<T>, grid, dim3(kThreads), 0, stream, a, part, DP,
                               static_cast<T*>(x.dk), static_cast<T*>(x.dv), cut);
            err = hipGetLastError();
            if (err != hipSuccess) return err;
        }
    }
    if (x.dbias != nullptr) {
        constexpr int type = sizeof(T) == 4 ? POINTOPS_F32 : __is_same(T, f16) ? POINTOPS_F16 : POINTOPS_BF16;
        return bucket_sums(a.bk, dbias_part, a.B, a.H, static_cast<int>(query_blocks), bias_entries(a.reach),
                           a.reach + kMargin, type, x.dbias, stream);
    }
    return hipSuccess;
}

template <typename T>
hipError_t backward(const Args& a, const Grads& x, hipStream_t stream) {
    const bool vec = vector_rows<T>(a.q, a.D) && vector_rows<T>(a.k, a.D) && vector_rows<T>(a.v, a.D) &&
                     vector_rows<T>(x.grad, a.D) && reinterpret_cast<uintptr_t>(x.out) % 16 == 0;
    return with_width(a.D, [&](auto width) {
        constexpr int DP = decltype(width)::value;
        return vec ? launch_backward<T, DP, true>(a, x, stream) : launch_backward<T, DP, false>(a, x, stream);
    });
}

}  // namespace
}  // namespace attn
}  // namespace pointops

extern "C" {

size_t pointops_attention_backward_workspace_bytes(const pointops_attention* in) {
    using namespace pointops::attn;
    Args a;
    return read_args(in, &a) ? workspace_of(a).bytes : 0;
}

hipError_t pointops_attention_backward(const pointops_attention* in, const void* out, const float* lse,
                                       const void* grad_out, const int64_t* grad_stride, void* dq, void* dk, void* dv,
                                       void* dbias, void* workspace, hipStream_t stream) {
    using namespace pointops::attn;
    Args a;
    if (!read_args(in, &a)) return hipErrorInvalidValue;
    if (a.B == 0 || a.H == 0 || (a.Q == 0 && a.N == 0)) return hipSuccess;
    if (dbias != nullptr && a.bias == nullptr) return hipErrorInvalidValue;
    if (a.Q > 0 && (in->q == nullptr || out == nullptr || lse == nullptr || grad_out == nullptr || grad_stride == nullptr ||
                    dq == nullptr || workspace == nullptr))
        return hipErrorInvalidValue;
    if (a.N > 0 && (in->k == nullptr || in->v == nullptr || dk == nullptr || dv == nullptr)) return hipErrorInvalidValue;
    Grads x{out, lse, {}, dq, dk, dv, dbias, static_cast<char*>(workspace)};
    if (grad_stride != nullptr) x.grad = {grad_out, grad_stride[0], grad_stride[1], grad_stride[2]};
    switch (in->type) {
        case POINTOPS_F32: return backward<float>(a, x, stream);
        case POINTOPS_F16: return backward<f16>(a, x, stream);
        default: return backward<bf16>(a, x, stream);
    }
}

}  // extern "C"
