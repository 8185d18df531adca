// Attention of one or a few new queries over what is kept: a sequence's own cache, in
// the tokens' type or in 8 or 4 bits, and a common start of the whole batch before it.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(s_ij - max_j s_ij) / sum,  s_ij = scale q_i k_j + bias(i - j)
//
// over the keys j that query i sees: positions 0 .. P - 1 are the start's, P + j the
// cache's.  The sum over j is cut into parts, each with its own maximum m, sum l and
// output o (32 bits); parts a and b join as o = o_a 2^(m_a - m) + o_b 2^(m_b - m), m = max,
// so that the start's part is one computation for all sequences: its rows are the queries
// of all of them, and its keys and values are read once.
//
// A wave takes 32 keys at a time for itself and 16 COLS rows (queries by heads of a
// key head) as columns of 16 x 16 products: keys straight from memory into the product's
// registers, values through the wave's own piece of LDS (for the transposing read),
// without a barrier in the loop.  Codes become bfloat16 on the way, two by an instruction
// with their scale and exactly; so queries over codes are held as the sum of 1 (bfloat16),
// 2 (float16) or 3 (float32) bfloat16 values, and weights as that of 2 or 3, and the
// products lose none of their bits.  Sixteen columns, not 32: a step of one token has H / G
// rows a key head, mostly 16 or fewer, and the products and exponentials of the columns
// that stay empty are work too.
#pragma once

#include <algorithm>

#include "quantized_cache.hpp"

namespace pointops {
namespace attn {

// Forms of keys and values.
enum Form { kAligned = 0, kAny = 1, kEight = 8, kFour = 4 };  // rows of 16-byte pieces, any rows, codes

// Keys and values of a sequence's cache or of the common start.  Strides of batch,
// token and head are in bytes, the scales' of batch and head.
struct Kept {
    const char *k, *v;
    const uint8_t *k_scales, *v_scales;
    int64_t kb, kn, kh, vb, vn, vh, sb, sh;
    int tokens;
};

struct CacheArgs {
    Rows q;
    bool q_vec;
    Kept own, start;
    const void *bias, *lengths;
    int B, Q, H, G, D;
    int window, sinks, reach, length_bits;
    float scale_log2;
    Buckets bk;

    __device__ __forceinline__ int length(int b) const {
        if (lengths == nullptr) return own.tokens;
        const int64_t l = length_bits == 64 ? static_cast<const int64_t*>(lengths)[b]
                                            : static_cast<const int32_t*>(lengths)[b];
        return static_cast<int>(l < 0 ? 0 : l > own.tokens ? own.tokens : l);
    }
};

constexpr int kStepWaves = 4, kStepThreads = kStepWaves * kWave;
constexpr int kKeys = 32;  // of a wave at a time

// Parts of a sum over keys: of a unit (key head with 16 COLS rows), `splits` of them,
// each `rows` long; a part is its maximum and its sum, two unused, then the values.
__host__ __device__ constexpr int part_width(int DP) { return DP + 4; }

struct CachePlan {
    int start_cols, own_cols;             // 16-row columns of a block
    int start_blocks, own_blocks;         // blocks of rows of a key head (of a sequence's key head)
    int start_splits, own_splits;         // 0: no start
    int64_t start_units, own_units;       // key heads by blocks of rows (by sequences)
    int64_t start_floats;                 // of the start's parts, ahead of the own ones
    bool direct;                          // one part: no join
};

// ------------------------------------------------------------ small pieces
template <typename T>
__device__ __forceinline__ f32x4 mma16(i32x4 a, i32x4 b, f32x4 acc) {
    if constexpr (sizeof(T) == 4) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], acc, 0, 0, 0);
        return acc;
    } else if constexpr (__is_same(T, bf16)) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
    }
}

// Over the four lanes of a column (l, l + 16, l + 32, l + 48).
__device__ __forceinline__ float quads_max(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(f2i(v), f2i(v), false, false);
    return halves_max(fmaxf(i2f(r[0]), i2f(r[1])));
}
__device__ __forceinline__ float quads_sum(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(f2i(v), f2i(v), false, false);
    return halves_sum(i2f(r[0]) + i2f(r[1]));
}

// What the products are computed in, and of how many values of it queries and weights
// are the sum.
template <typename T, int FORM>
struct Products {
    static constexpr bool kCoded = FORM == kEight || FORM == kFour;
    using C = std::conditional_t<kCoded, bf16, T>;
    static constexpr int kQuery = !kCoded ? 1 : sizeof(T) == 4 ? 3 : __is_same(T, f16) ? 2 : 1;
    static constexpr int kWeight = sizeof(T) == 2 ? 2 : kCoded ? 3 : 1;
};

// x as N fragments of C that add up to it.
template <typename C, int N>
__device__ __forceinline__ void split(const float* x, i32x4 (&out)[N]) {
    float left[kPerFrag<C>];
#pragma unroll
    for (int e = 0; e < kPerFrag<C>; ++e) left[e] = x[e];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        out[n] = as_fragment<C>(left);
        if (n + 1 < N) {
#pragma unroll
            for (int e = 0; e < kPerFrag<C>; ++e) {
                const float taken = element<C>(out[n], e);
                left[e] = finite(taken) ? left[e] - taken : 0.f;
            }
        }
    }
}

// ------------------------------------------------- 32 keys on their way in
// Fragment c of a row's values: lane l holds those from column(c, l / 16) on.  Codes come
// 16 (64 columns of the row's four lanes) at a time, the last 32 columns 8.
template <typename T, int FORM, int DP>
struct Incoming {
    using C = typename Products<T, FORM>::C;
    static constexpr bool kCoded = Products<T, FORM>::kCoded;
    static constexpr int kFrags = DP * static_cast<int>(sizeof(C)) / 64;  // of a key's row
    using TileT = Tile<C, DP>;
    static constexpr int kTileBytes = kKeys * TileT::kStride;

    __device__ static __forceinline__ int column(int c, int quad) {
        if constexpr (!kCoded) return (4 * c + quad) * kPerFrag<C>;
        else return c < DP / 64 * 2 ? c / 2 * 64 + quad * 16 + c % 2 * 8 : c * 32 + quad * 8;
    }

    // ---- rows of a type
    static constexpr int kPerRow = DP * static_cast<int>(sizeof(C)) / 16;      // 16-byte pieces
    static constexpr int kPieces = kKeys * kPerRow / kWave;
    // ---- codes: words of eight, pieces of 16 values
    static constexpr int kWords = FORM == kEight ? 2 : 1;
    static constexpr int kCodePerRow = DP / 16, kCodePieces = kKeys * kCodePerRow / kWave;
    static constexpr int kRowBytes = FORM == kEight ? DP : DP / 2, kScales = DP / kGroup;

    i32x4 kr[kCoded ? 1 : 2][kCoded ? 1 : kFrags], vr[kCoded ? 1 : kPieces];
    uint32_t kc[kCoded ? 2 : 1][kCoded ? kFrags * kWords : 1], vc[kCoded ? kCodePieces : 1][kCoded ? 2 * kWords : 1];
    uint32_t ks[kCoded ? 2 : 1][kCoded ? kScales : 1], vs[kCoded ? kCodePieces : 1];

    template <int N>
    __device__ static __forceinline__ void words(const uint8_t* p, uint32_t* out) {
        if constexpr (N == 4) {
            const i32x4 x = *reinterpret_cast<const i32x4*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = x[i];
        } else if constexpr (N == 2) {
            const i32x2 x = *reinterpret_cast<const i32x2*>(p);
            out[0] = x[0];
            out[1] = x[1];
        } else {
            out[0] = *reinterpret_cast<const uint32_t*>(p);
        }
    }

    // Keys j0 .. j0 + 31 of the head at k and v; from `limit` (>= 1) on the last one again, for which
    // the caller's scores are masked.
    __device__ __forceinline__ void load(const Kept& kept, const char* k, const char* v, const uint8_t* k_scales,
                                         const uint8_t* v_scales, int j0, int limit, int width) {
        const int lane = lane_id(), col = lane % 16, quad = lane / 16;
        if constexpr (!kCoded) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const T* const row = reinterpret_cast<const T*>(k + min(j0 + 16 * u + col, limit - 1) * kept.kn);
#pragma unroll
                for (int c = 0; c < kFrags; ++c) kr[u][c] = load_row<T, FORM == kAligned>(row, column(c, quad), width);
            }
#pragma unroll
            for (int x = 0; x < kPieces; ++x) {
                const int at = x * kWave + lane;
                const T* const row = reinterpret_cast<const T*>(v + min(j0 + at / kPerRow, limit - 1) * kept.vn);
                vr[x] = load_row<T, FORM == kAligned>(row, at % kPerRow * kPerFrag<T>, width);
            }
        } else {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int64_t j = min(j0 + 16 * u + col, limit - 1);
                const uint8_t* const row = reinterpret_cast<const uint8_t*>(k) + j * kRowBytes;
#pragma unroll
                for (int c = 0; c + 1 < kFrags; c += 2) words<2 * kWords>(row + column(c, quad) * kWords / 2, kc[u] + c * kWords);
                if constexpr (kFrags % 2 != 0)
                    words<kWords>(row + column(kFrags - 1, quad) * kWords / 2, kc[u] + (kFrags - 1) * kWords);
                load_scales(k_scales + j * kScales, ks[u]);
            }
#pragma unroll
            for (int x = 0; x < kCodePieces; ++x) {
                const int at = x * kWave + lane, piece = at % kCodePerRow;
                const int64_t j = min(j0 + at / kCodePerRow, limit - 1);
                words<2 * kWords>(reinterpret_cast<const uint8_t*>(v) + j * kRowBytes + piece * 8 * kWords, vc[x]);
                vs[x] = v_scales[j * kScales + piece / 2];
            }
        }
    }
    // The scales of a row's groups, as bytes in one word or (96 values) one by one.
    __device__ static __forceinline__ void load_scales(const uint8_t* p, uint32_t* out) {
        if constexpr (kScales == 4) {
            const uint32_t x = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = x >> (8 * i) & 255;
        } else if constexpr (kScales == 2) {
            const uint32_t x = *reinterpret_cast<const uint16_t*>(p);
            out[0] = x & 255;
            out[1] = x >> 8;
        } else {
#pragma unroll
            for (int i = 0; i < kScales; ++i) out[i] = p[i];
        }
    }

    // Row operand: keys 16 u + lane % 16, fragment c.
    __device__ __forceinline__ i32x4 keys(int u, int c) const {
        if constexpr (!kCoded) {
            return kr[u][c];
        } else {
            const int quad = lane_id() / 16;
            const uint32_t byte = c < DP / 64 * 2 ? (quad < 2 ? ks[u][c / 2 * 2] : ks[u][c / 2 * 2 + 1]) : ks[u][c];
            return decode8<FORM>(kc[u] + c * kWords, scale_of(byte));
        }
    }

    __device__ __forceinline__ void store_values(char* tile) const {
        const int lane = lane_id();
        if constexpr (!kCoded) {
#pragma unroll
            for (int x = 0; x < kPieces; ++x) {
                const int at = x * kWave + lane;
                *reinterpret_cast<i32x4*>(tile + at / kPerRow * TileT::kStride + at % kPerRow * 16) = vr[x];
            }
        } else {
#pragma unroll
            for (int x = 0; x < kCodePieces; ++x) {
                const int at = x * kWave + lane;
                i32x4* const to = reinterpret_cast<i32x4*>(tile + at / kCodePerRow * TileT::kStride + at % kCodePerRow * 32);
                const float scale = scale_of(vs[x]);
                to[0] = decode8<FORM>(vc[x], scale);
                to[1] = decode8<FORM>(vc[x] + kWords, scale);
            }
        }
    }

    // Transposed operand: its row is column 16 d + lane % 16 of the tile, its values keys
    // 16 u + 4 (lane / 16) + e: of both halves u for 16 bits (the order of two results'
    // registers), of half u for 32.
    __device__ static __forceinline__ i32x4 values(const char* tile, int u, int d) {
        const int lane = lane_id(), i = lane % 16, quad = lane / 16;
        if constexpr (sizeof(C) == 4) {
            const char* p = tile + (16 * u + 4 * quad) * TileT::kStride + 4 * (16 * d + i);
            i32x4 r;
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = *reinterpret_cast<const int*>(p + e * TileT::kStride);
            return r;
        } else {
            const char* p = tile + (4 * quad + i / 4) * TileT::kStride + 2 * (16 * d + 4 * (i % 4));
            typedef __attribute__((address_space(3))) s16x4 lds4;
            const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p));
            const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 16 * TileT::kStride));
            const i32x2 a = __builtin_bit_cast(i32x2, x), b = __builtin_bit_cast(i32x2, y);
            return i32x4{a[0], a[1], b[0], b[1]};
        }
    }
};

// ------------------------------------------------------------ careful rows
// One query by a whole wave, key by key, for rows whose sums are not finite: there a
// product with a masked key's infinity or NaN may have spread.  Lane l holds elements l
// and l + 64.
template <typename T, int FORM>
struct CarefulKept {
    float q0, q1, m = -kInf, l = 0.f, o0 = 0.f, o1 = 0.f;
    bool d0, d1;
    float scale_log2;

    __device__ __forceinline__ CarefulKept(const CacheArgs& a, const T* q) : scale_log2(a.scale_log2) {
        const int lane = lane_id();
        d0 = lane < a.D;
        d1 = lane + kWave < a.D;
        q0 = d0 ? to_float(q[lane]) : 0.f;
        q1 = d1 ? to_float(q[lane + kWave]) : 0.f;
    }
    __device__ static __forceinline__ float value(const char* row, const uint8_t* scales, int at) {
        if constexpr (FORM == kEight || FORM == kFour) return decode_one<FORM>(reinterpret_cast<const uint8_t*>(row), scales, at);
        else return to_float(reinterpret_cast<const T*>(row)[at]);
    }
    __device__ __forceinline__ void add(const char* k, const char* v, const uint8_t* ks, const uint8_t* vs, float bias) {
        if (bias == -kInf) return;
        const int lane = lane_id();
        const float s = wave_sum((d0 ? q0 * value(k, ks, lane) : 0.f) + (d1 ? q1 * value(k, ks, lane + kWave) : 0.f)) * scale_log2 + bias;
        if (s == -kInf) return;
        const float top = fmaxf(m, s), keep = m == -kInf ? 0.f : exp2_fast(m - top), w = exp2_fast(s - top);
        m = top;
        l = l * keep + w;
        o0 = o0 * keep + (d0 ? w * value(v, vs, lane) : 0.f);
        o1 = o1 * keep + (d1 ? w * value(v, vs, lane + kWave) : 0.f);
    }
    __device__ __forceinline__ bool settled(bool n0, bool n1) const {
        return ballot((n0 && finite(o0)) || (n1 && finite(o1))) == 0;
    }
};

// ------------------------------------------------------------------ a part
template <int COLS, int DP>
constexpr int kSumBytes = 16 * COLS * (DP + 4) * 4;
// The waves' tiles, then their sums in the same place; maxima and sums of the weights; then
// the bias: [buckets][heads of the rows], the buckets of 0 .. reach, the edges.
template <typename T, int FORM, int DP, int COLS>
constexpr int kTilesBytes = kStepWaves * Incoming<T, FORM, DP>::kTileBytes > kSumBytes<COLS, DP>
                                ? kStepWaves * Incoming<T, FORM, DP>::kTileBytes : kSumBytes<COLS, DP>;
template <typename T, int FORM, int DP, int COLS>
constexpr int kStepLds = kTilesBytes<T, FORM, DP, COLS> + 2 * kStepWaves * 16 * COLS * 4;
inline int bias_heads(int group, int cols) { return group < 16 * cols ? group : 16 * cols; }
constexpr size_t bias_most(int cols) { return 4 * (256 * 16 * cols) + (kMaxReach + 4) / 4 * 4 + 4 * 255; }
inline size_t bias_lds(const CacheArgs& a, int cols) {
    if (a.bias == nullptr) return 0;
    return 4 * static_cast<size_t>(a.bk.count) * bias_heads(a.H / a.G, cols) + (a.reach + 4) / 4 * 4 + 4 * a.bk.n;
}

// Keys of `kept` that the query at position p sees: as Seen, in the kept keys' own numbers.
__device__ __forceinline__ Seen seen_of(const CacheArgs& a, int p, int base, int limit) {
    if (p < 0) return {0, 0, 0};
    const int low = max(0, p - a.window + 1 - base), high = min(p - base, limit - 1);
    return {low, max(0, high - low + 1), max(0, min(min(a.sinks, p + 1) - base, limit))};
}

// One block's part of one unit.  START: the common start (rows of all sequences), else the
// cache of sequence b.
template <typename T, int FORM, int DP, int COLS, bool START>
__device__ __forceinline__ void attention_part(const CacheArgs& a, T* __restrict__ out, float* __restrict__ part, int b0,
                                               int g, int r0, int split_at, int splits, char* lds) {
    using In = Incoming<T, FORM, DP>;
    using C = typename In::C;
    constexpr int kQ = Products<T, FORM>::kQuery, kW = Products<T, FORM>::kWeight, kFrags = In::kFrags;
    constexpr int kOut = DP / 16, kSumStride = DP + 4, kRows = 16 * COLS;
    const Kept& kept = START ? a.start : a.own;
    const int lane = lane_id(), col = lane % 16, quad = lane / 16, wave = uniform(threadIdx.x / kWave);
    const int group = a.H / a.G, per = a.Q * group, total = START ? a.B * per : per;
    const int rows = min(kRows, total - r0), base = START ? 0 : a.start.tokens;
    float* const tops = reinterpret_cast<float*>(lds + kTilesBytes<T, FORM, DP, COLS>);
    float* const totals = tops + kStepWaves * kRows;
    float* const table = totals + kStepWaves * kRows;

    // Rows: this lane's columns.
    const int own_length = START ? 0 : uniform(a.length(b0));
    const int limit = START ? kept.tokens : own_length;
    int p[COLS];
    Seen seen[COLS];
    int first = 0, low = INT32_MAX, high = -1, low_most = 0, high_least = INT32_MAX, p_least = INT32_MAX;
#pragma unroll
    for (int n = 0; n < COLS; ++n) {
        const int r = r0 + 16 * n + col;
        const bool mine = 16 * n + col < rows;
        p[n] = -1;
        if (mine) {
            const int length = START ? a.length(r / per) : own_length;
            p[n] = a.start.tokens + length - a.Q + (START ? r % per : r) / group;
        }
        seen[n] = seen_of(a, p[n], base, limit);
        first = max(first, seen[n].first);
        if (seen[n].count > 0) {
            low = min(low, seen[n].low);
            high = max(high, seen[n].low + seen[n].count - 1);
        }
        if (mine) {
            // (A row that sees nothing of these is masked in every tile.)
            low_most = max(low_most, seen[n].low);
            high_least = min(high_least, seen[n].low + seen[n].count - 1);
            p_least = min(p_least, p[n]);
        }
    }
    first = wave_max_i32_l63(first);
    low = -wave_max_i32_l63(-low);
    high = wave_max_i32_l63(high);
    low_most = wave_max_i32_l63(low_most);
    high_least = -wave_max_i32_l63(-high_least);
    p_least = -wave_max_i32_l63(-p_least);
    // Tiles of keys: the first keys', then the window's.
    const int first_tiles = (first + kKeys - 1) / kKeys;
    const int low_tile = high < 0 ? first_tiles : max(first_tiles, low / kKeys);
    const int tiles = first_tiles + max(0, (high < 0 ? 0 : high / kKeys + 1) - low_tile);
    const int begin = static_cast<int>(static_cast<int64_t>(tiles) * split_at / splits);
    const int end = static_cast<int>(static_cast<int64_t>(tiles) * (split_at + 1) / splits);
    auto first_key = [&](int tile) { return (tile < first_tiles ? tile : tile - first_tiles + low_tile) * kKeys; };

    const int64_t b = START ? 0 : b0;
    const char* const k = kept.k + b * kept.kb + g * kept.kh;
    const char* const v = kept.v + b * kept.vb + g * kept.vh;
    const uint8_t* const k_scales = kept.k_scales + b * kept.sb + g * kept.sh;
    const uint8_t* const v_scales = kept.v_scales + b * kept.sb + g * kept.sh;
    In in;
    int tile = begin + wave;
    if (tile < end) in.load(kept, k, v, k_scales, v_scales, first_key(tile), limit, a.D);

    i32x4 q[COLS][kFrags][kQ];
#pragma unroll
    for (int n = 0; n < COLS; ++n) {
        const int r = r0 + 16 * n + col, in_b = START ? r % per : r;
        const bool mine = 16 * n + col < rows;
        const T* const row = a.q.at<T>(START ? r / per : b0, g * group + in_b % group) + in_b / group * a.q.n;
#pragma unroll
        for (int c = 0; c < kFrags; ++c) {
            const int at = In::column(c, quad);
            float x[kPerFrag<C>];
#pragma unroll
            for (int e = 0; e < kPerFrag<C>; ++e) x[e] = 0.f;
            if (mine) {
                if (a.q_vec) {
#pragma unroll
                    for (int e = 0; e < kPerFrag<C>; e += kPerFrag<T>) {
                        const i32x4 piece = load_row<T, true>(row, at + e, a.D);
#pragma unroll
                        for (int f = 0; f < kPerFrag<T>; ++f) x[e + f] = element<T>(piece, f);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < kPerFrag<C>; ++e)
                        if (at + e < a.D) x[e] = to_float(row[at + e]);
                }
            }
            split<C, kQ>(x, q[n][c]);
        }
    }

    const bool biased = a.bias != nullptr;
    const int heads = min(group, kRows);
    uint8_t* const ids = reinterpret_cast<uint8_t*>(table + a.bk.count * heads);
    int head[COLS];  // this lane's columns' heads in the table
    float far[COLS];
    if (biased) {
        int* const edges = reinterpret_cast<int*>(ids + (a.reach + 4) / 4 * 4);
        for (int x = threadIdx.x; x < a.bk.n; x += kStepThreads) edges[x] = a.bk.edge[x];
        const int h0 = g * group + (heads < group ? r0 % group : 0);
        for (int x = threadIdx.x; x < a.bk.count * heads; x += kStepThreads) {
            const int h = heads < group ? g * group + (r0 + x % heads) % group : h0 + x % heads;
            table[x] = bias_log2(to_float(static_cast<const T*>(a.bias)[static_cast<int64_t>(x / heads) * a.H + h]));
        }
        __syncthreads();
        for (int x = threadIdx.x; x <= a.reach; x += kStepThreads) ids[x] = static_cast<uint8_t>(bucket_of(a.bk, edges, x));
        __syncthreads();
#pragma unroll
        for (int n = 0; n < COLS; ++n) {
            head[n] = heads < group ? 16 * n + col : (r0 + 16 * n + col) % group;
            far[n] = table[a.bk.n * heads + head[n]];
        }
    }
    auto bias_at = [&](int offset, int column) { return table[ids[min(max(offset, 0), a.reach)] * heads + column]; };

    // Scores as the products leave them, in units of 1 / factor: a bias needs them scaled,
    // and a negative scale turns their order.
    const bool scaled = biased || !(a.scale_log2 > 0.f);
    const float factor = scaled ? 1.f : a.scale_log2;
    char* const values = lds + wave * In::kTileBytes;
    f32x4 o[kOut][COLS];
    float m[COLS], l[COLS];
#pragma unroll
    for (int n = 0; n < COLS; ++n) {
        m[n] = -kInf;
        l[n] = 0.f;
#pragma unroll
        for (int d = 0; d < kOut; ++d) o[d][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (; tile < end; tile += kStepWaves) {
        const int j0 = first_key(tile);
        f32x4 s[COLS][2];
#pragma unroll
        for (int n = 0; n < COLS; ++n) s[n][0] = s[n][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kFrags; ++c)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const i32x4 f = in.keys(u, c);
#pragma unroll
                for (int n = 0; n < COLS; ++n)
#pragma unroll
                    for (int x = 0; x < kQ; ++x) s[n][u] = mma16<C>(f, q[n][c][x], s[n][u]);
            }
        in.store_values(values);
        if (tile + kStepWaves < end) in.load(kept, k, v, k_scales, v_scales, first_key(tile + kStepWaves), limit, a.D);
        const bool whole = j0 >= low_most && j0 + kKeys - 1 <= high_least;
        const bool all_far = p_least - (base + j0 + kKeys - 1) >= a.reach;
        i32x4 w[COLS][8 / kPerFrag<C>][kW];
#pragma unroll
        for (int n = 0; n < COLS; ++n) {
            float x[8];  // keys 16 u + 4 quad + e, as u, e
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = scaled ? s[n][e / 4][e % 4] * a.scale_log2 : s[n][e / 4][e % 4];
            const int j = j0 + 4 * quad;
            if (biased) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] += all_far ? far[n] : bias_at(p[n] - base - (j + e / 4 * 16 + e % 4), head[n]);
            }
            if (!whole) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (!seen[n](j + e / 4 * 16 + e % 4)) x[e] = -kInf;
            }
            float top = x[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) top = fmaxf(top, x[e]);
            top = quads_max(top) * factor;
            if (ballot(top > m[n] + kSlack) != 0) {
                const float next = fmaxf(m[n], top);
                const float keep = m[n] == next ? 1.f : exp2_fast(m[n] - next);
                m[n] = next;
                l[n] *= keep;
#pragma unroll
                for (int d = 0; d < kOut; ++d) o[d][n] *= keep;
            }
            const float less = m[n] == -kInf ? 0.f : m[n];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = exp2_fast(__builtin_fmaf(x[e], factor, -less));
                l[n] += x[e];
            }
#pragma unroll
            for (int f = 0; f < 8 / kPerFrag<C>; ++f) split<C, kW>(x + f * kPerFrag<C>, w[n][f]);
        }
        lanes_exchange();
#pragma unroll
        for (int d = 0; d < kOut; ++d)
#pragma unroll
            for (int f = 0; f < 8 / kPerFrag<C>; ++f) {
                const i32x4 x = In::values(values, f, d);
#pragma unroll
                for (int n = 0; n < COLS; ++n)
#pragma unroll
                    for (int y = 0; y < kW; ++y) o[d][n] = mma16<C>(x, w[n][f][y], o[d][n]);
            }
        lanes_exchange();
    }

    // The waves' parts, brought to their common maximum and added in order.
    float mine_by[COLS];
#pragma unroll
    for (int n = 0; n < COLS; ++n) {
        l[n] = quads_sum(l[n]);
        if (quad == 0) {
            tops[wave * kRows + 16 * n + col] = m[n];
            totals[wave * kRows + 16 * n + col] = l[n];
        }
    }
    __syncthreads();  // also: the tiles' LDS is free
    float top[COLS], sum[COLS];
#pragma unroll
    for (int n = 0; n < COLS; ++n) {
        top[n] = tops[16 * n + col];
#pragma unroll
        for (int x = 1; x < kStepWaves; ++x) top[n] = fmaxf(top[n], tops[x * kRows + 16 * n + col]);
        const float less = top[n] == -kInf ? 0.f : top[n];
        sum[n] = 0.f;
#pragma unroll
        for (int x = 0; x < kStepWaves; ++x) sum[n] += totals[x * kRows + 16 * n + col] * exp2_fast(tops[x * kRows + 16 * n + col] - less);
        mine_by[n] = exp2_fast(m[n] - less);
    }
    float* const sums = reinterpret_cast<float*>(lds);
    for (int x = 0; x < kStepWaves; ++x) {
        if (x == wave) {
#pragma unroll
            for (int n = 0; n < COLS; ++n)
#pragma unroll
                for (int d = 0; d < kOut; ++d) {
                    f32x4* const at = reinterpret_cast<f32x4*>(sums + (16 * n + col) * kSumStride + 16 * d + 4 * quad);
                    f32x4 y = x == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : *at;
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(o[d][n][e], mine_by[n], y[e]);
                    *at = y;
                }
        }
        __syncthreads();
    }
    if (quad == 0 && wave == 0) {
#pragma unroll
        for (int n = 0; n < COLS; ++n) {
            tops[16 * n + col] = top[n];
            totals[16 * n + col] = sum[n];
        }
    }
    __syncthreads();
    // Rows of the block, one a wave at a time: out, or the split's part of it.
    for (int row = wave; row < rows; row += kStepWaves) {
        const int r = r0 + row, in_b = START ? r % per : r, bb = START ? r / per : b0;
        const int i = in_b / group, h = g * group + in_b % group;
        float x0 = lane < a.D ? sums[row * kSumStride + lane] : 0.f;
        float x1 = lane + kWave < a.D ? sums[row * kSumStride + lane + kWave] : 0.f;
        float lm = tops[row], ll = totals[row];
        // A sum of weights that is NaN comes from a seen pair, and all of its row is NaN as it
        // lies, but where a bias of -inf masks that pair.
        const bool none = ll != ll;
        const int column = heads < group ? row : in_b % group;
        bool masks = false;
        if (none && biased)
            for (int x = lane; x < a.bk.count; x += kWave) masks |= table[x * heads + column] == -kInf;
        const bool n0 = none || !finite(x0), n1 = none || !finite(x1);
        if (ll == 0.f) {
            x0 = x1 = 0.f;
        } else if (none ? ballot(masks) != 0 : ballot(n0 || n1) != 0) {
            CarefulKept<T, FORM> c(a, a.q.at<T>(bb, h) + i * a.q.n);
            const int at = a.start.tokens + (START ? uniform(a.length(bb)) : own_length) - a.Q + i;
            const Seen sees = seen_of(a, at, base, limit);
            bool done = false;
            for (int t = begin; t < end && !done; ++t)
                for (int j = first_key(t); j < first_key(t) + kKeys && !done; ++j)
                    if (sees(j)) {
                        const int64_t n = j;
                        c.add(k + n * kept.kn, v + n * kept.vn, k_scales + n * In::kScales, v_scales + n * In::kScales,
                              biased ? bias_at(at - base - j, column) : 0.f);
                        done = none ? c.l != c.l : c.settled(n0, n1);
                    }
            if (none) {
                lm = c.m;
                ll = c.l;
            }
            // To the maximum of the products' sums.
            const float by = none ? 1.f : exp2_fast(c.m - lm);
            x0 = n0 ? c.o0 * by : x0;
            x1 = n1 ? c.o1 * by : x1;
        }
        if (part == nullptr) {
            const float inv = ll == 0.f ? 0.f : 1.f / ll;
            T* const dst = out + ((static_cast<int64_t>(bb) * a.Q + i) * a.H + h) * a.D;
            if (lane < a.D) dst[lane] = from_float<T>(x0 * inv);
            if (lane + kWave < a.D) dst[lane + kWave] = from_float<T>(x1 * inv);
        } else {
            float* const dst = part + static_cast<int64_t>(row) * part_width(DP);
            if (lane == 0) {
                dst[0] = lm;
                dst[1] = ll;
            }
            if (lane < a.D) dst[4 + lane] = x0;
            if (lane + kWave < a.D) dst[4 + lane + kWave] = x1;
        }
    }
}

// The start's blocks, then the caches'.
template <typename T, int FORM, int DP, int START_COLS, int OWN_COLS>
__global__ __launch_bounds__(kStepThreads, START_COLS > 1 || OWN_COLS > 1 || sizeof(T) == 4 ? 1 : 2) void attention_cache_kernel(
    const CacheArgs a, const CachePlan plan, T* __restrict__ out, float* __restrict__ parts) {
    extern __shared__ __attribute__((aligned(16))) char cache_lds[];
    const int64_t block = blockIdx.x, start = plan.start_units * plan.start_splits;
    if (block < start) {
        const int split_at = static_cast<int>(block % plan.start_splits);
        const int unit = static_cast<int>(block / plan.start_splits);
        attention_part<T, FORM, DP, START_COLS, true>(
            a, out, parts + block * (16 * START_COLS) * part_width(DP), 0, unit / plan.start_blocks,
            unit % plan.start_blocks * (16 * START_COLS), split_at, plan.start_splits, cache_lds);
    } else {
        const int64_t at = block - start;
        const int split_at = static_cast<int>(at % plan.own_splits);
        const int64_t unit = at / plan.own_splits, bg = unit / plan.own_blocks;
        attention_part<T, FORM, DP, OWN_COLS, false>(
            a, out, plan.direct ? nullptr : parts + plan.start_floats + at * (16 * OWN_COLS) * part_width(DP),
            static_cast<int>(bg / a.G), static_cast<int>(bg % a.G), static_cast<int>(unit % plan.own_blocks) * (16 * OWN_COLS),
            split_at, plan.own_splits, cache_lds);
    }
}

// Columns of 16 rows that one wave takes at once where there are more than 16 rows: as
// many as its registers hold.
constexpr int kManyCols = 2;

template <typename T, int FORM>
hipError_t launch_cache_form(const CacheArgs& a, const CachePlan& plan, void* out, float* parts, hipStream_t stream) {
    constexpr int M = kManyCols;
    const int64_t blocks = plan.start_units * plan.start_splits + plan.own_units * plan.own_splits;
    return with_width(a.D, [&](auto width) {
        constexpr int DP = decltype(width)::value;
        const int which = plan.start_cols == 1 ? 0 : plan.own_cols == 1 ? 1 : 2;
        auto* kernel = attention_cache_kernel<T, FORM, DP, M, M>;
        if constexpr (FORM != kAny) {  // (whose plans have no others)
            if (which == 0) kernel = attention_cache_kernel<T, FORM, DP, 1, 1>;
            if (which == 1) kernel = attention_cache_kernel<T, FORM, DP, M, 1>;
        }
        const size_t one = kStepLds<T, FORM, DP, 1> + bias_lds(a, 1), many = kStepLds<T, FORM, DP, M> + bias_lds(a, M);
        const size_t lds = which == 0 ? one : which == 1 ? std::max(one, many) : many;
        if (lds > kLdsFree) {
            static std::atomic<uint64_t> allowed[3];
            const size_t most = std::max(kStepLds<T, FORM, DP, 1> + bias_most(1), kStepLds<T, FORM, DP, M> + bias_most(M));
            const hipError_t err = allow_lds(kernel, allowed[which], most);
            if (err != hipSuccess) return err;
        }
        hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(blocks)), dim3(kStepThreads), lds, stream, a, plan,
                           static_cast<T*>(out), parts);
        return hipGetLastError();
    });
}

}  // namespace attn
}  // namespace pointops
