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
//
// A long cache's keys are bound by HBM: 4 x 65536 tokens of 32 heads over 8 of 128 in 8 bits 73 us,
// 6.0 TB/s; in 4 bits under float16 by what two waves a SIMD issue between their waits (32 x 8192: 47
// us, 4.6 TB/s; vector instructions 40 % of the time, LDS 39, matrix units 25); the start's rows by
// what is issued beside the products (64 sequences behind 65536 tokens: 455 to 470 T/s of the pairs,
// matrix units 40 % busy); short ones by one block's latency (10 to 18 us).
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

// Division of 0 .. 2^31 - 1 by a number of the call, as a product and a shift (a division
// by what the compiler does not know is some thirty instructions, and a row asks for several), as by
// Granlund and Montgomery, "Division by invariant integers using multiplication" (1994):
// n / d = (n m / 2^32 + n) / 2^s with s = ceil(log2 d), m = floor(2^32 (2^s - d) / d) + 1.
struct Divisor {
    uint32_t d, m, s;
    static Divisor of(int64_t d) {
        uint32_t s = 0;
        while ((int64_t(1) << s) < d) ++s;
        return {static_cast<uint32_t>(d), static_cast<uint32_t>((((uint64_t(1) << s) - d) << 32) / d + 1), s};
    }
    __device__ __forceinline__ int of_row(int n) const {
        return static_cast<int>((__umulhi(static_cast<uint32_t>(n), m) + static_cast<uint32_t>(n)) >> s);
    }
};

struct CacheArgs {
    Divisor group, per;  // heads of a key head, rows of a sequence's key head (those by its queries)
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
// The running maximum may lie 8 (in units of log 2; float16: 3) below the true one.
template <typename C>
constexpr float kMostWeight = static_cast<float>(1 << static_cast<int>(kMostLog<C>));
constexpr size_t kMostLds = 160 * 1024;

// Parts of a sum over keys: of a unit (a key head with a block of rows), `splits` of them,
// each `rows` long; a part is its maximum and its sum, two unused, then the values.
__host__ __device__ constexpr int part_width(int DP) { return DP + 4; }

struct Parts {
    // A part's rows (of a block's 2^shift those that there are, where it is the only one), blocks of
    // rows of a key head, parts of each (0: none).
    int rows, shift, blocks, splits;
    int64_t units;                    // key heads (the caches': of all sequences) by blocks of rows
    int64_t floats;
    __device__ __forceinline__ const float* first(const float* parts, int head, int row, int width) const {
        const int64_t unit = static_cast<int64_t>(head) * blocks + (row >> shift);
        return parts + (unit * splits * rows + (row & ((1 << shift) - 1))) * width;
    }
};

struct CachePlan {
    int shape;         // of Shape
    Parts start, own;  // the caches' parts lie behind the start's
    bool joined;       // a launch of its own joins the parts
};

// ------------------------------------------------------------ small pieces
// acc += A B of 32 values of 16 bits, or step e of four of 16 values of 32 bits.  An instruction
// waits for the one before it on the same registers: the callers take two or four sums in turn.
template <typename T>
constexpr int kMmaSteps = sizeof(T) == 4 ? 4 : 1;
template <typename T>
__device__ __forceinline__ f32x4 mma16(i32x4 a, i32x4 b, f32x4 acc, int e) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4, a)[e], __builtin_bit_cast(f32x4, b)[e], acc, 0, 0, 0);
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

// Two values rounded to C in one word.
template <typename C>
__device__ __forceinline__ int pair_of(float x, float y) {
    if constexpr (__is_same(C, bf16)) {
        return __builtin_bit_cast(int, __builtin_convertvector((f32x2{x, y}), bf16x2));
    } else {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(int, __builtin_convertvector((f32x2{x, y}), f16x2));
    }
}
template <typename C>
__device__ __forceinline__ float half_of(int pair, int which) {
    if constexpr (__is_same(C, bf16)) return i2f(which == 0 ? pair << 16 : pair & static_cast<int>(0xffff0000u));
    else return static_cast<float>(__builtin_bit_cast(f16, static_cast<uint16_t>(which == 0 ? pair : pair >> 16)));
}

// x as N fragments of C that add up to it (of an infinity, FINITE: all but the first are NaN).
template <typename C, int N, bool FINITE>
__device__ __forceinline__ void split(const float* x, i32x4 (&out)[N]) {
    if constexpr (sizeof(C) == 4) {
        out[0] = as_fragment<C>(x);
    } else {
        float left[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) left[e] = x[e];
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                out[n][i] = pair_of<C>(left[2 * i], left[2 * i + 1]);
#pragma unroll
                for (int e = 2 * i; n + 1 < N && e < 2 * i + 2; ++e) {
                    const float taken = half_of<C>(out[n][i], e % 2);
                    left[e] = FINITE || finite(taken) ? left[e] - taken : 0.f;
                }
            }
    }
}

// Buffer loads of what is read once and in whole lines: it does not stay in the caches.
// Of a wave's own values (32 heads over 8 of 128, all loads kept: 64 x 2048 bfloat16 tokens 103 us,
// values alone past the caches 82, keys too, of whose lines a load takes the half, 93;
// 4 x 65536 in 8 bits 108, 90, 94; 32 x 8192 in 4 bits, float16, 55, 55, 60).
constexpr int kOnce = 2;
// An offset behind every buffer: reads there give zeros and touch nothing.
constexpr uint32_t kNothing = 0x80000000u;
// A value that stays in its register: left to itself the compiler chooses between two
// offsets by a branch at every load, each with a wait for the loads before.
__device__ __forceinline__ uint32_t fixed(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
}
// `rows` rows (of `bytes` each, at least one) from j0 on of those at `base`, as a buffer that ends with
// the last.  A tile of rows lies within 2 GiB.
__device__ __forceinline__ auto rows_from(const void* base, uint32_t stride, int j0, int rows, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(static_cast<const char*>(base) + static_cast<uint64_t>(static_cast<uint32_t>(j0)) * stride), 0,
        static_cast<int>(static_cast<uint32_t>(rows - 1) * stride) + bytes, kRawBuffer);
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
    static constexpr bool kWhole = FORM == kFour && DP == 128;  // a row's four lanes hold a group of 32 each

    __device__ static __forceinline__ int column(int c, int quad) {
        if constexpr (!kCoded) return (4 * c + quad) * kPerFrag<C>;
        else if constexpr (kWhole) return quad * 32 + c * 8;
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
    uint32_t ks[kCoded ? 2 : 1], vs[kCoded ? kCodePieces : 1];

    // Offsets of this lane's pieces in a tile: of its key in either half, of its first value
    // and (rows of 96 values) its others, of scales; what lies behind a row's width: kNothing.
    static constexpr int kVectors = kCoded ? kCodePieces : kPieces, kVectorsPerRow = kCoded ? kCodePerRow : kPerRow;
    static constexpr bool kSteps = kWave % kVectorsPerRow == 0;  // a lane's values are in one column
    uint32_t k_at[2], v_at[kSteps ? 1 : kVectors], ks_at[kCoded ? 2 : 1], vs_at[!kCoded ? 1 : kSteps ? 1 : kVectors];
    uint32_t behind;  // of the last 32 columns of a key's row: kNothing in a lane past the width, else 0 (a bit each of two)

    __device__ __forceinline__ void set(const Kept& kept, int width) {
        const int lane = lane_id(), col = lane % 16, quad = lane / 16;
        const uint32_t kn = kCoded ? kRowBytes : static_cast<uint32_t>(kept.kn), vn = kCoded ? kRowBytes : static_cast<uint32_t>(kept.vn);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            k_at[u] = fixed((16 * u + col) * kn + (kCoded ? column(0, quad) * kWords / 2 : 16 * quad));
            if constexpr (kCoded) ks_at[u] = fixed((16 * u + col) * kScales);
        }
#pragma unroll
        for (int x = 0; x < (kSteps ? 1 : kVectors); ++x) {
            const uint32_t at = x * kWave + lane, row = at / kVectorsPerRow, piece = at % kVectorsPerRow;
            const bool past = !kCoded && static_cast<int>(piece) * kPerFrag<T> >= width;
            v_at[x] = fixed(past ? kNothing : row * vn + piece * (kCoded ? 8 * kWords : 16));
            if constexpr (kCoded) vs_at[x] = fixed(row * kScales + piece / 2);
        }
        if constexpr (!kCoded) {
            behind = 0;
#pragma unroll
            for (int c = kFrags - kLast; c < kFrags; ++c)
                if (column(c, quad) >= width) behind |= kNothing >> (kFrags - 1 - c);
            behind = fixed(behind);
        }
    }
    static constexpr int kLast = static_cast<int>(sizeof(C)) / 2;  // fragments of 32 columns

    // Keys j0 .. j0 + 31 of the head at k and v; zeros from `limit` (> j0) on, for which the
    // caller's scores are masked.
    __device__ __forceinline__ void load(const Kept& kept, const char* k, const char* v, const uint8_t* k_scales,
                                         const uint8_t* v_scales, int j0, int limit, int width) {
        const int lane = lane_id(), col = lane % 16, quad = lane / 16;
        if constexpr (FORM == kAny) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int j = min(j0 + 16 * u + col, limit - 1);
#pragma unroll
                for (int c = 0; c < kFrags; ++c) kr[u][c] = load_row<T, false>(reinterpret_cast<const T*>(k + j * kept.kn), column(c, quad), width);
            }
#pragma unroll
            for (int x = 0; x < kPieces; ++x) {
                const int at = x * kWave + lane, j = min(j0 + at / kPerRow, limit - 1);
                vr[x] = load_row<T, false>(reinterpret_cast<const T*>(v + j * kept.vn), at % kPerRow * kPerFrag<T>, width);
            }
        } else if constexpr (FORM == kAligned) {
            const int rows = min(limit - j0, kKeys), bytes = width * static_cast<int>(sizeof(T));
            const auto ks = rows_from(k, static_cast<uint32_t>(kept.kn), j0, rows, bytes);
            const auto vs = rows_from(v, static_cast<uint32_t>(kept.vn), j0, rows, bytes);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int c = 0; c < kFrags; ++c) {
                    const uint32_t past = c < kFrags - kLast ? 0 : behind << (kFrags - 1 - c) & kNothing;
                    kr[u][c] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(ks, (k_at[u] + 64 * c) | past, 0, 0));
                }
#pragma unroll
            for (int x = 0; x < kPieces; ++x)
                vr[x] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(
                    vs, kSteps ? v_at[0] + x * (kWave / kPerRow) * static_cast<uint32_t>(kept.vn) : v_at[x], 0, kOnce));
        } else {
            const int rows = min(limit - j0, kKeys);
            const auto k0 = rows_from(k, kRowBytes, j0, rows, kRowBytes), v0 = rows_from(v, kRowBytes, j0, rows, kRowBytes);
            const auto ks0 = rows_from(k_scales, kScales, j0, rows, kScales), vs0 = rows_from(v_scales, kScales, j0, rows, kScales);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if constexpr (kWhole) words<4, 0>(k0, k_at[u], kc[u]);
                else {
#pragma unroll
                    for (int c = 0; c + 1 < kFrags; c += 2) words<2 * kWords, 0>(k0, k_at[u] + c * 16 * kWords, kc[u] + c * kWords);
                }
                // (The last 32 columns: eight a lane, not sixteen.)
                if constexpr (kFrags % 2 != 0)
                    words<kWords, 0>(k0, k_at[u] + (column(kFrags - 1, quad) - (kFrags > 1 ? column(0, quad) : quad * 8)) * kWords / 2,
                                  kc[u] + (kFrags - 1) * kWords);
                ks[u] = scale_bytes(ks0, ks_at[u]);
            }
#pragma unroll
            for (int x = 0; x < kCodePieces; ++x) {
                words<2 * kWords, kOnce>(v0, kSteps ? v_at[0] + x * (kWave / kCodePerRow) * kRowBytes : v_at[x], vc[x]);
                vs[x] = __builtin_amdgcn_raw_buffer_load_b8(vs0, kSteps ? vs_at[0] + x * (kWave / kCodePerRow) * kScales : vs_at[x], 0, 0);
            }
        }
    }
    template <int N, int POLICY, typename R>
    __device__ static __forceinline__ void words(R rows, uint32_t at, uint32_t* out) {
        if constexpr (N == 4) {
            const i32x4 x = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rows, at, 0, POLICY));
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = x[i];
        } else if constexpr (N == 2) {
            const i32x2 x = __builtin_bit_cast(i32x2, __builtin_amdgcn_raw_buffer_load_b64(rows, at, 0, POLICY));
            out[0] = x[0];
            out[1] = x[1];
        } else {
            out[0] = __builtin_amdgcn_raw_buffer_load_b32(rows, at, 0, POLICY);
        }
    }
    // The scales of a row's groups, a byte each.
    template <typename R>
    __device__ static __forceinline__ uint32_t scale_bytes(R rows, uint32_t at) {
        if constexpr (kScales == 4) return __builtin_amdgcn_raw_buffer_load_b32(rows, at, 0, 0);
        else if constexpr (kScales == 2) return static_cast<uint16_t>(__builtin_amdgcn_raw_buffer_load_b16(rows, at, 0, 0));
        else if constexpr (kScales == 1) return static_cast<uint8_t>(__builtin_amdgcn_raw_buffer_load_b8(rows, at, 0, 0));
        else {
            uint32_t all = 0;
#pragma unroll
            for (int i = 0; i < kScales; ++i)
                all |= static_cast<uint32_t>(static_cast<uint8_t>(__builtin_amdgcn_raw_buffer_load_b8(rows, at + i, 0, 0))) << (8 * i);
            return all;
        }
    }

    // Row operand: keys 16 u + lane % 16, fragment c.
    __device__ __forceinline__ i32x4 keys(int u, int c) const {
        if constexpr (!kCoded) {
            return kr[u][c];
        } else {
            const int group = kWhole ? lane_id() / 16 : c < DP / 64 * 2 ? c / 2 * 2 + lane_id() / 32 : c;
            return decode8<FORM>(kc[u] + c * kWords, scale_of(ks[u] >> (8 * group) & 255));
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
// product with a masked key's infinity or NaN may have spread, or their finite values have
// passed 32 bits (the weights reach 2^8 and their number).
template <typename T, int FORM>
struct CarefulKept : CarefulSum {
    float q0, q1;
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
        CarefulSum::add(s, d0 ? value(v, vs, lane) : 0.f, d1 ? value(v, vs, lane + kWave) : 0.f);
    }
};

// ------------------------------------------------- keys that waves share
// 32 KW keys and values of the common start on their way through a block's registers to
// LDS, where its waves read both.  Rows behind `limit` are zeros (a descriptor that ends
// with the last row), for which the caller's scores are masked.
template <typename T, int FORM, int DP, int KW, int THREADS>
struct Shared {
    using C = typename Products<T, FORM>::C;
    static constexpr bool kCoded = Products<T, FORM>::kCoded;
    using TileT = Tile<C, DP>;
    static constexpr int kRows = kKeys * KW, kBytes = 2 * kRows * TileT::kStride;
    static constexpr int kPerRow = kCoded ? DP / 16 : DP * static_cast<int>(sizeof(C)) / 16;
    static constexpr int kPieces = (kRows * kPerRow + THREADS - 1) / THREADS;
    static constexpr bool kAll = kRows * kPerRow % THREADS == 0;
    static constexpr int kWords = FORM == kEight ? 2 : 1, kRowBytes = FORM == kEight ? DP : DP / 2, kScales = DP / kGroup;
    static constexpr int kPieceBytes = kCoded ? 8 * kWords : 16;
    i32x4 r[2][kPieces];
    uint32_t scale[kCoded ? 2 : 1][kCoded ? kPieces : 1];

    uint32_t at[2][kPieces], scale_at[kCoded ? kPieces : 1];

    __device__ __forceinline__ void set(const Kept& kept, int width) {
#pragma unroll
        for (int side = 0; side < 2; ++side)
#pragma unroll
            for (int x = 0; x < kPieces; ++x) {
                const uint32_t stride = kCoded ? kRowBytes : static_cast<uint32_t>(side == 0 ? kept.kn : kept.vn);
                const uint32_t n = x * THREADS + threadIdx.x, row = n / kPerRow, piece = n % kPerRow;
                const bool here = (kAll || row < kRows) && (kCoded || static_cast<int>(piece) * kPerFrag<T> < width);
                at[side][x] = fixed(here ? row * stride + piece * kPieceBytes : kNothing);
                if constexpr (kCoded)
                    if (side == 0) scale_at[x] = fixed(here ? row * kScales + piece / 2 : kNothing);
            }
    }
    __device__ __forceinline__ void load(const Kept& kept, const char* k, const char* v, const uint8_t* k_scales,
                                         const uint8_t* v_scales, int j0, int limit, int width) {
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const int count = min(limit - j0, kRows);
            const auto rows = rows_from(side == 0 ? k : v, kCoded ? kRowBytes : static_cast<uint32_t>(side == 0 ? kept.kn : kept.vn), j0,
                                        count, kCoded ? kRowBytes : width * static_cast<int>(sizeof(T)));
#pragma unroll
            for (int x = 0; x < kPieces; ++x) {
                if constexpr (kPieceBytes == 16) r[side][x] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rows, at[side][x], 0, 0));
                else {
                    const i32x2 y = __builtin_bit_cast(i32x2, __builtin_amdgcn_raw_buffer_load_b64(rows, at[side][x], 0, 0));
                    r[side][x] = i32x4{y[0], y[1], 0, 0};
                }
            }
            if constexpr (kCoded) {
                const auto scales = rows_from(side == 0 ? k_scales : v_scales, kScales, j0, count, kScales);
#pragma unroll
                for (int x = 0; x < kPieces; ++x) scale[side][x] = __builtin_amdgcn_raw_buffer_load_b8(scales, scale_at[x], 0, 0);
            }
        }
    }
    // Keys, then values.
    __device__ __forceinline__ void store(char* tiles) const {
#pragma unroll
        for (int side = 0; side < 2; ++side)
#pragma unroll
            for (int x = 0; x < kPieces; ++x) {
                const int at = x * THREADS + static_cast<int>(threadIdx.x), row = at / kPerRow;
                if (!kAll && row >= kRows) continue;
                i32x4* const to = reinterpret_cast<i32x4*>(tiles + (side * kRows + row) * TileT::kStride + at % kPerRow * (kCoded ? 32 : 16));
                if constexpr (kCoded) {
                    const uint32_t codes[4] = {static_cast<uint32_t>(r[side][x][0]), static_cast<uint32_t>(r[side][x][1]),
                                               static_cast<uint32_t>(r[side][x][2]), static_cast<uint32_t>(r[side][x][3])};
                    to[0] = decode8<FORM>(codes, scale_of(scale[side][x]));
                    to[1] = decode8<FORM>(codes + kWords, scale_of(scale[side][x]));
                } else {
                    to[0] = r[side][x];
                }
            }
    }
    // Row operand: key `row` + lane % 16 of those in LDS, fragment c: values from column(c, lane / 16) on.
    __device__ static __forceinline__ int column(int c, int quad) { return (4 * c + quad) * kPerFrag<C>; }
    __device__ static __forceinline__ i32x4 keys(const char* tiles, int row, int c) {
        const int lane = lane_id();
        return *reinterpret_cast<const i32x4*>(tiles + (row + lane % 16) * TileT::kStride + 64 * c + 16 * (lane / 16));
    }
};

// The same for rows of 16 bits, which memory loads write to LDS themselves: 64 lanes' pieces of
// 16 bytes one behind the other, so that rows have no room between them.  Each lane asks for the
// piece that belongs there: within a row, piece p lies at p ^ turn(row), with which 8 neighbouring
// rows of a row operand's read lie in 8 different places of 128 bytes, and the 4 rows and 2 pieces of a
// transposing read too.  (Rows of 256 bytes have 16 places, of which these are one half, and rows 8
// apart share them: counters call half of LDS's time conflicts.)  What lies
// behind a row's width is cleared once; loads past the descriptor's end bring zeros.
// 64 sequences behind 65536 tokens of width 128, in turn: 167 us through registers, 146 to 151 so (LDS
// instructions 15 to 6 % of the time, the matrix units 37 to 40 % busy); 32 behind 32768 of width
// 96 37 and 35, of 64 30 to 31 either way.
template <typename T, int DP, int KW, int WAVES>
struct Streamed {
    static constexpr int kRows = kKeys * KW, kRowBytes = DP * 2, kPerRow = DP / 8, kBytes = 2 * kRows * kRowBytes;
    static constexpr int kLoads = kRows * kPerRow / kWave / WAVES;  // of a wave and side, 1 KB each
    static_assert(kRows * kPerRow % (kWave * WAVES) == 0);
    // Pieces change places among 8 where rows are a multiple of 128 bytes, among 4 in others.
    __device__ static __forceinline__ uint32_t turn(uint32_t row) {
        if constexpr (kPerRow % 8 == 0) return (row & 3) << 1 | (row >> 2 & 1);
        else return (row >> 1 & 1) << 1 | (row >> 2 & 1);
    }
    uint32_t at[2][kLoads];  // of this lane's pieces in a tile of rows; kNothing: none
    uint32_t key_at[2], value_at[4];
    int wave;

    __device__ __forceinline__ uint32_t row_of(int x) const { return (static_cast<uint32_t>(x * WAVES + wave) * kWave + lane_id()) / kPerRow; }
    __device__ __forceinline__ uint32_t piece_of(int x) const {
        const uint32_t n = static_cast<uint32_t>(x * WAVES + wave) * kWave + lane_id();
        return n % kPerRow ^ turn(n / kPerRow);
    }
    __device__ __forceinline__ void set(const Kept& kept, int width) {
        wave = uniform(threadIdx.x / kWave);
        const uint32_t lane = lane_id(), col = lane % 16, quad = lane / 16;
#pragma unroll
        for (int x = 0; x < kLoads; ++x) {
            const bool here = static_cast<int>(piece_of(x)) * 8 < width;
            at[0][x] = fixed(here ? row_of(x) * static_cast<uint32_t>(kept.kn) + piece_of(x) * 16 : kNothing);
            at[1][x] = fixed(here ? row_of(x) * static_cast<uint32_t>(kept.vn) + piece_of(x) * 16 : kNothing);
        }
        // Key lane % 16's piece 4 c + quad, of even and of odd c.
        const uint32_t turned = turn(col), high = turned / 4 * 64;
        key_at[0] = col * kRowBytes + (quad ^ turned % 4) * 16 + high;
        key_at[1] = col * kRowBytes + (quad ^ turned % 4) * 16 - high;
        // Of keys 4 quad + i / 4 (i = lane % 16) columns 16 d + 4 (i % 4) .. + 3, of d % 4 = 0 .. 3.
        const uint32_t row = 4 * quad + col / 4, by = turn(row);
#pragma unroll
        for (uint32_t d = 0; d < 4; ++d)
            value_at[d] = row * kRowBytes + (d ^ by / 2) * 32 + (col % 4 / 2 ^ by % 2) * 16 + col % 2 * 8;
    }
    template <typename Rows>
    __device__ static __forceinline__ void bring(Rows rows, char* to, uint32_t from) {
        typedef __attribute__((address_space(3))) void lds_t;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rows, (lds_t*)to, 16, from, 0, 0, 0);
    }
    __device__ __forceinline__ void load(const Kept& kept, const char* k, const char* v, int j0, int limit, int width, char* tiles) const {
        const int count = min(limit - j0, kRows), bytes = width * 2;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const uint32_t stride = static_cast<uint32_t>(side == 0 ? kept.kn : kept.vn);
            const auto rows = rows_from(side == 0 ? k : v, stride, j0, count, bytes);
            char* const to = tiles + side * kRows * kRowBytes + wave * (kWave * 16);
            if (count == kRows) {
#pragma unroll
                for (int x = 0; x < kLoads; ++x) bring(rows, to + x * WAVES * kWave * 16, at[side][x]);
            } else {
#pragma unroll
                for (int x = 0; x < kLoads; ++x) {
                    // Behind the last row: that row again (its scores are masked).
                    const uint32_t row = min(row_of(x), static_cast<uint32_t>(count - 1));
                    bring(rows, to + x * WAVES * kWave * 16, at[side][x] == kNothing ? kNothing : row * stride + piece_of(x) * 16);
                }
            }
        }
    }
    // What this wave has asked for lies in LDS (vmcnt 0, the other counters left alone).
    __device__ __forceinline__ void arrived() const { __builtin_amdgcn_s_waitcnt(0x0f70); }
    // Row operand: key `row` + lane % 16 (row a multiple of 16), fragment c.
    __device__ __forceinline__ i32x4 keys(const char* tiles, int row, int c) const {
        return *reinterpret_cast<const i32x4*>(tiles + row * kRowBytes + 64 * c + key_at[c % 2]);
    }
    // Transposed operand of the 32 keys from `row` on: Incoming's order.
    __device__ __forceinline__ i32x4 values(const char* tiles, int row, int d) const {
        const char* const p = tiles + (kRows + row) * kRowBytes + d / 4 * 128 + value_at[d % 4];
        typedef __attribute__((address_space(3))) s16x4 lds4;
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p));
        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 16 * kRowBytes));
        const i32x2 a = __builtin_bit_cast(i32x2, x), b = __builtin_bit_cast(i32x2, y);
        return i32x4{a[0], a[1], b[0], b[1]};
    }
};

// ------------------------------------------------------------- joining parts
// A row's sum over keys, in a wave: lane l holds values l and l + 64.  All are 2^-above of
// what they are by the maximum m.
struct RowSum {
    float m = -kInf, l = 0.f, x0 = 0.f, x1 = 0.f, above = 0.f;

    // Adds `count` parts, `step` floats from one to the next, in order.
    __device__ __forceinline__ void add(const float* first, int64_t step, int count, int D) {
        if (count == 0) return;
        const int lane = lane_id(), c0 = 4 + min(lane, D - 1), c1 = 4 + min(lane + kWave, D - 1);
        constexpr int kAtOnce = 16;
        float y0[kAtOnce], y1[kAtOnce];
        auto ask = [&](int from) {  // (past the end: the last one again, for which the factor is not used)
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                const float* const at = first + min(from + k, count - 1) * step;
                y0[k] = at[c0];
                y1[k] = at[c1];
            }
        };
        ask(0);  // (beside the maxima)
        float top = -kInf;
        for (int s = lane; s < count; s += kWave) top = fmaxf(top, first[s * step]);
        top = fmaxf(m, wave_max(top));
        const float less = top == -kInf ? 0.f : top, keep = exp2_fast(m - less);
        m = top;
        x0 *= keep;
        x1 *= keep;
        float sum = 0.f;
        for (int from = 0; from < count; from += kWave) {
            // A lane's part: its factor; then the parts' rows one after another.
            const int s = from + lane;
            float by = 0.f;
            if (s < count) {
                by = exp2_fast(first[s * step] - less - above);
                sum = __builtin_fmaf(first[s * step + 1], by, sum);
            }
            const int some = min(kWave, count - from);
            for (int i = 0; i < some; i += kAtOnce) {
                if (from + i > 0) ask(from + i);
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) {
                    if (i + k < some) {
                        const float f = i2f(readlane(f2i(by), i + k));
                        x0 = __builtin_fmaf(y0[k], f, x0);
                        x1 = __builtin_fmaf(y1[k], f, x1);
                    }
                }
            }
        }
        l = __builtin_fmaf(l, keep, wave_sum(sum));
    }
    // The means.
    __device__ __forceinline__ void divide() {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        x0 *= inv;
        x1 *= inv;
    }
    template <typename T>
    __device__ __forceinline__ void write(T* dst, int D) const {
        const int lane = lane_id();
        if (lane < D) dst[lane] = from_float<T>(x0);
        if (lane + kWave < D) dst[lane + kWave] = from_float<T>(x1);
    }
};

// ------------------------------------------------------------------ a part
// The rows and keys of a block: the common start with rows of all sequences, a sequence's
// cache with its rows, or its rows with both, one behind the other.
enum Kind { kStart, kOwn, kBoth };

// A block's waves: ROW_WAVES hold 16 COLS rows each, and so many of them share 32 keys at
// a time; 1: every wave has the same rows and takes its own keys.
template <typename T, int FORM, int DP, int COLS, int ROW_WAVES, int WAVES>
struct StepLds {
    static constexpr int kKeyWaves = WAVES / ROW_WAVES, kRows = 16 * COLS * ROW_WAVES;
    static constexpr int kSums = kRows * (DP + 4) * 4;
    static constexpr bool kStreamed = ROW_WAVES > 1 && FORM == kAligned && sizeof(T) == 2;
    static constexpr int kTiles = ROW_WAVES == 1 ? WAVES * Incoming<T, FORM, DP>::kTileBytes
                                  : kStreamed    ? 2 * Streamed<T, DP, kKeyWaves, WAVES>::kBytes
                                                 : 2 * Shared<T, FORM, DP, kKeyWaves, kWave * WAVES>::kBytes;
    // The tiles, then the sums in the same place; maxima and sums of the weights; then the
    // bias: [buckets][heads of the rows], the buckets of 0 .. reach, the edges.
    static constexpr int kPlace = kTiles > kSums ? kTiles : kSums;
    static constexpr int kBytes = kPlace + 2 * kKeyWaves * kRows * 4;
};
inline size_t bias_lds(const CacheArgs& a, int rows) {
    if (a.bias == nullptr) return 0;
    return 4 * static_cast<size_t>(a.bk.count) * std::min(a.H / a.G, rows) + (a.reach + 4) / 4 * 4 + 4 * a.bk.n;
}

// Keys of `kept` that the query at position p sees: as Seen, in the kept keys' own numbers.
__device__ __forceinline__ Seen seen_of(const CacheArgs& a, int p, int base, int limit) {
    if (p < 0) return {0, 0, 0};
    const int low = max(0, p - a.window + 1 - base), high = min(p - base, limit - 1);
    return {low, max(0, high - low + 1), max(0, min(min(a.sinks, p + 1) - base, limit))};
}

// What a block reads of one of the kept: keys 0 .. limit - 1 at positions `base` on, of
// which its rows see the first `first_tiles` tiles and those from `low_tile` on.
template <int TILE, int COLS>
struct Range {
    const Kept* kept;
    const char *k, *v;
    const uint8_t *k_scales, *v_scales;
    int base, limit, first_tiles, low_tile, tiles;
    int low_most, high_least;  // keys in between are seen by all of the wave's rows
    Seen seen[COLS];

    __device__ __forceinline__ int first_key(int tile) const {
        return (tile < first_tiles ? tile : tile - first_tiles + low_tile) * TILE;
    }
    __device__ __forceinline__ void tiles_of(int first, int low, int high) {
        first_tiles = (first + TILE - 1) / TILE;
        low_tile = high < 0 ? first_tiles : max(first_tiles, low / TILE);
        tiles = first_tiles + max(0, (high < 0 ? 0 : high / TILE + 1) - low_tile);
    }
};

// One block's part of one unit.
template <typename T, int FORM, int DP, int COLS, int ROW_WAVES, int WAVES, int KIND>
__device__ __forceinline__ void attention_part(const CacheArgs& a, T* __restrict__ out, float* __restrict__ part, int b0,
                                               int g, int r0, int split_at, int splits, char* lds) {
    using Lds = StepLds<T, FORM, DP, COLS, ROW_WAVES, WAVES>;
    constexpr int kKeyWaves = Lds::kKeyWaves, kRows = Lds::kRows, kThreads = kWave * WAVES;
    constexpr bool kShared = ROW_WAVES > 1, kManySequences = KIND == kStart, kStreamed = Lds::kStreamed;
    using In = Incoming<T, FORM, DP>;
    using Sh = Shared<T, FORM, DP, kKeyWaves, kWave * WAVES>;
    using C = typename In::C;
    constexpr int kQ = Products<T, FORM>::kQuery, kW = Products<T, FORM>::kWeight, kFrags = In::kFrags;
    constexpr int kOut = DP / 16, kSumStride = DP + 4, kTile = kShared ? kKeys * kKeyWaves : kKeys;
    constexpr int kRanges = KIND == kBoth ? 2 : 1;
    const int lane = lane_id(), col = lane % 16, quad = lane / 16, wave = uniform(threadIdx.x / kWave);
    const int row_wave = wave % ROW_WAVES, key_wave = wave / ROW_WAVES;
    const int w0 = 16 * COLS * row_wave;  // this wave's first row in the block
    const int group = a.group.d, per = a.per.d, total = kManySequences ? a.B * per : per;
    // A row's sequence, query and head in the group.
    struct Row {
        int b, i, h;
    };
    auto row_of = [&](int r) {
        const int b = kManySequences ? a.per.of_row(r) : b0, in = kManySequences ? r - b * per : r, i = a.group.of_row(in);
        return Row{b, i, in - i * group};
    };
    const int rows = min(kRows, total - r0);
    float* const tops = reinterpret_cast<float*>(lds + Lds::kPlace);
    float* const totals = tops + kKeyWaves * kRows;
    float* const table = totals + kKeyWaves * kRows;

    // Rows: this lane's columns.
    const int own_length = kManySequences ? 0 : uniform(a.length(b0));
    Row mine[COLS];
    int p[COLS], p_least = INT32_MAX;
#pragma unroll
    for (int n = 0; n < COLS; ++n) {
        // (Columns without a row: the block's first, whose values they do not read.)
        const bool any = w0 + 16 * n + col < rows;
        mine[n] = row_of(any ? r0 + w0 + 16 * n + col : r0);
        p[n] = -1;
        if (any) {
            p[n] = a.start.tokens + (kManySequences ? a.length(mine[n].b) : own_length) - a.Q + mine[n].i;
            p_least = min(p_least, p[n]);
        }
    }
    p_least = -wave_max_i32_l63(-p_least);
    Range<kTile, COLS> range[kRanges];
#pragma unroll
    for (int x = 0; x < kRanges; ++x) {
        Range<kTile, COLS>& at = range[x];
        const bool start = KIND == kStart || (KIND == kBoth && x == 0);
        at.kept = start ? &a.start : &a.own;
        at.base = start ? 0 : a.start.tokens;
        at.limit = start ? a.start.tokens : own_length;
        const int64_t b = start ? 0 : b0;
        at.k = at.kept->k + b * at.kept->kb + g * at.kept->kh;
        at.v = at.kept->v + b * at.kept->vb + g * at.kept->vh;
        at.k_scales = at.kept->k_scales + b * at.kept->sb + g * at.kept->sh;
        at.v_scales = at.kept->v_scales + b * at.kept->sb + g * at.kept->sh;
        int first = 0, low = INT32_MAX, high = -1, low_most = 0, high_least = INT32_MAX;
#pragma unroll
        for (int n = 0; n < COLS; ++n) {
            const Seen seen = seen_of(a, p[n], at.base, at.limit);
            at.seen[n] = seen;
            first = max(first, seen.first);
            if (seen.count > 0) {
                low = min(low, seen.low);
                high = max(high, seen.low + seen.count - 1);
            }
            if (w0 + 16 * n + col < rows) {
                // (A row that sees nothing of these is masked in every tile.)
                low_most = max(low_most, seen.low);
                high_least = min(high_least, seen.low + seen.count - 1);
            }
        }
        first = wave_max_i32_l63(first);
        low = -wave_max_i32_l63(-low);
        high = wave_max_i32_l63(high);
        at.low_most = wave_max_i32_l63(low_most);
        at.high_least = -wave_max_i32_l63(-high_least);
        if constexpr (kShared) {
            // What any of the block's rows sees.
            int* const ends = reinterpret_cast<int*>(tops);
            if (lane == 0) {
                ends[3 * wave] = first;
                ends[3 * wave + 1] = low;
                ends[3 * wave + 2] = high;
            }
            __syncthreads();
#pragma unroll
            for (int y = 0; y < WAVES; ++y) {
                first = max(first, ends[3 * y]);
                low = min(low, ends[3 * y + 1]);
                high = max(high, ends[3 * y + 2]);
            }
            first = uniform(first);
            low = uniform(low);
            high = uniform(high);
            __syncthreads();
        }
        at.tiles_of(first, low, high);
    }
    const int first_range = range[0].tiles, tiles = kRanges == 2 ? first_range + range[kRanges - 1].tiles : first_range;
    // The first `over` parts have one tile more.
    const int each = tiles / splits, over = tiles - each * splits;
    const int begin = split_at * each + min(split_at, over), end = begin + each + (split_at < over ? 1 : 0);
    std::conditional_t<kStreamed, Streamed<T, DP, kKeyWaves, WAVES>, std::conditional_t<kShared, Sh, In>> in;
    in.set(*range[0].kept, a.D);
    bool in_second = false;
    auto fetch = [&](int tile, char* to) {
        const bool second = kRanges == 2 && tile >= first_range;
        const Range<kTile, COLS>& at = range[second ? kRanges - 1 : 0];
        if (second && !in_second) {  // (whose strides may be others)
            in.set(*at.kept, a.D);
            in_second = true;
        }
        const int from = at.first_key(second ? tile - first_range : tile);
        if constexpr (kStreamed) in.load(*at.kept, at.k, at.v, from, at.limit, a.D, to);
        else in.load(*at.kept, at.k, at.v, at.k_scales, at.v_scales, from, at.limit, a.D);
    };
    int tile = kShared ? begin : begin + wave;
    if constexpr (kStreamed) {
        if (a.D < DP) {
            for (int x = threadIdx.x; x < Lds::kTiles / 16; x += kThreads) reinterpret_cast<i32x4*>(lds)[x] = i32x4{0, 0, 0, 0};
            __syncthreads();
        }
    }
    if (tile < end) fetch(tile, lds);

    i32x4 q[COLS][kFrags][kQ];
#pragma unroll
    for (int n = 0; n < COLS; ++n) {
        const bool any = w0 + 16 * n + col < rows;
        const T* const row = a.q.at<T>(mine[n].b, g * group + mine[n].h) + mine[n].i * a.q.n;
#pragma unroll
        for (int c = 0; c < kFrags; ++c) {
            const int at = kShared ? Sh::column(c, quad) : In::column(c, quad);
            float x[kPerFrag<C>];
#pragma unroll
            for (int e = 0; e < kPerFrag<C>; ++e) x[e] = 0.f;
            if (any) {
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
            split<C, kQ, false>(x, q[n][c]);
        }
    }

    const bool biased = a.bias != nullptr;
    const int heads = min(group, kRows);
    uint8_t* const ids = reinterpret_cast<uint8_t*>(table + a.bk.count * heads);
    int head[COLS];  // this lane's columns' heads in the table
    float far[COLS];
    if (biased) {
        int* const edges = reinterpret_cast<int*>(ids + (a.reach + 4) / 4 * 4);
        for (int x = threadIdx.x; x < a.bk.n; x += kThreads) edges[x] = a.bk.edge[x];
        for (int x = threadIdx.x; x < a.bk.count * heads; x += kThreads) {
            const int at = x % heads, in = r0 + at - a.group.of_row(r0 + at) * group;
            const int h = g * group + (heads < group ? in : at);
            table[x] = bias_log2(to_float(static_cast<const T*>(a.bias)[static_cast<int64_t>(x / heads) * a.H + h]));
        }
        __syncthreads();
        for (int x = threadIdx.x; x <= a.reach; x += kThreads) ids[x] = static_cast<uint8_t>(bucket_of(a.bk, edges, x));
        __syncthreads();
#pragma unroll
        for (int n = 0; n < COLS; ++n) {
            head[n] = heads < group ? w0 + 16 * n + col : mine[n].h;
            far[n] = table[a.bk.n * heads + head[n]];
        }
    }
    auto bias_at = [&](int offset, int column) { return table[ids[min(max(offset, 0), a.reach)] * heads + column]; };

    // Scores as the products leave them, in units of 1 / factor: a bias needs them scaled,
    // and a negative scale turns their order.
    const bool scaled = biased || !(a.scale_log2 > 0.f);
    const float factor = scaled ? 1.f : a.scale_log2;
    f32x4 o[kOut][COLS];
    float m[COLS], l[COLS];
#pragma unroll
    for (int n = 0; n < COLS; ++n) {
        // (A row that sees nothing needs no maximum: its weights are zeros by any.)
        bool sees = false;
#pragma unroll
        for (int x = 0; x < kRanges; ++x) sees |= range[x].seen[n].count > 0 || range[x].seen[n].first > 0;
        m[n] = sees ? -kInf : 0.f;
        l[n] = 0.f;
#pragma unroll
        for (int d = 0; d < kOut; ++d) o[d][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    f32x4 s[COLS][2];
    i32x4 w[COLS][8 / kPerFrag<C>][kW];
    auto score = [&](auto&& keys) {
#pragma unroll
        for (int n = 0; n < COLS; ++n) s[n][0] = s[n][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kFrags; ++c) {
            const i32x4 f[2] = {keys(0, c), keys(1, c)};
#pragma unroll
            for (int x = 0; x < kQ; ++x)
#pragma unroll
                for (int e = 0; e < kMmaSteps<C>; ++e)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int n = 0; n < COLS; ++n) s[n][u] = mma16<C>(f[u], q[n][c][x], s[n][u], e);
        }
    };
    // Of the 32 keys from j0 on.
    auto weigh = [&](const Range<kTile, COLS>& at, int j0) {
        const int j = j0 + 4 * quad;  // register e of half u: key j + 16 u + e
        if (scaled) {
#pragma unroll
            for (int n = 0; n < COLS; ++n)
#pragma unroll
                for (int u = 0; u < 2; ++u) s[n][u] *= a.scale_log2;
        }
        if (biased) {
            if (p_least - (at.base + j0 + kKeys - 1) >= a.reach) {
#pragma unroll
                for (int n = 0; n < COLS; ++n)
#pragma unroll
                    for (int u = 0; u < 2; ++u) s[n][u] += far[n];
            } else {
#pragma unroll
                for (int n = 0; n < COLS; ++n)
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[n][e / 4][e % 4] += bias_at(p[n] - at.base - (j + e / 4 * 16 + e % 4), head[n]);
            }
        }
        if (j0 < at.low_most || j0 + kKeys - 1 > at.high_least) {
#pragma unroll
            for (int n = 0; n < COLS; ++n)
#pragma unroll
                for (int e = 0; e < 8; ++e) s[n][e / 4][e % 4] = at.seen[n](j + e / 4 * 16 + e % 4) ? s[n][e / 4][e % 4] : -kInf;
        }
        float x[COLS][8];
        auto form = [&]() {
#pragma unroll
            for (int n = 0; n < COLS; ++n) {
                const float less = m[n] == -kInf ? 0.f : m[n];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[n][e] = exp2_fast(__builtin_fmaf(s[n][e / 4][e % 4], factor, -less));
            }
        };
        // The weights by the maximum so far (its reference, in m); where one of them has outgrown
        // it (or there is none yet), by a new one.  So the scores' own maximum is seldom asked for.
        form();
        bool rises = false;
#pragma unroll
        for (int n = 0; n < COLS; ++n) {
            float most = x[n][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) most = fmaxf(most, x[n][e]);
            rises |= most > kMostWeight<C> || m[n] == -kInf;
        }
        if (ballot(rises) != 0) {
#pragma unroll
            for (int n = 0; n < COLS; ++n) {
                float top = s[n][0][0];
#pragma unroll
                for (int e = 1; e < 8; ++e) top = fmaxf(top, s[n][e / 4][e % 4]);
                const float next = fmaxf(m[n], reference_of<C>(quads_max(top) * factor));
                const float keep = m[n] == next ? 1.f : exp2_fast(m[n] - next);
                m[n] = next;
                l[n] *= keep;
#pragma unroll
                for (int d = 0; d < kOut; ++d) o[d][n] *= keep;
            }
            form();
        }
#pragma unroll
        for (int n = 0; n < COLS; ++n) {
            l[n] += ((x[n][0] + x[n][1]) + (x[n][2] + x[n][3])) + ((x[n][4] + x[n][5]) + (x[n][6] + x[n][7]));
#pragma unroll
            for (int f = 0; f < 8 / kPerFrag<C>; ++f) split<C, kW, true>(x[n] + f * kPerFrag<C>, w[n][f]);
        }
    };
    // The values' operands are read a batch ahead of their products, the first before the
    // weights are formed.
    constexpr int kHalves = 8 / kPerFrag<C>, kBatch = 2;
    static_assert(kOut % kBatch == 0);
    i32x4 vf[2][kBatch][kHalves];
    auto ask = [&](const char* values, int d, i32x4 (&f)[kBatch][kHalves]) {
#pragma unroll
        for (int x = 0; x < kBatch; ++x)
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                if constexpr (kStreamed) f[x][h] = in.values(values, kKeys * key_wave, d + x);
                else f[x][h] = In::values(values, h, d + x);
            }
    };
    auto add = [&](const char* values) {
#pragma unroll
        for (int d = 0; d < kOut; d += kBatch) {
            const auto& f = vf[d / kBatch % 2];
            if (d + kBatch < kOut) ask(values, d + kBatch, vf[(d / kBatch + 1) % 2]);
            keep_order();
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
#pragma unroll
                for (int y = 0; y < kW; ++y)
#pragma unroll
                    for (int e = 0; e < kMmaSteps<C>; ++e)
#pragma unroll
                        for (int x = 0; x < kBatch; ++x)
#pragma unroll
                            for (int n = 0; n < COLS; ++n) o[d + x][n] = mma16<C>(f[x][h], w[n][h][y], o[d + x][n], e);
        }
    };
    if constexpr (kShared) {
        // Two sets of tiles in LDS: one barrier a tile.
        constexpr int kSet = Lds::kTiles / 2;
        char* now = lds;
        if constexpr (kStreamed) in.arrived();
        else if (tile < end) in.store(now);
        __syncthreads();
        for (; tile < end; ++tile) {
            char* const then = now == lds ? lds + kSet : lds;
            if (tile + 1 < end) fetch(tile + 1, then);
            const int at = kKeys * key_wave;
            const char* const values = kStreamed ? now : now + (Sh::kRows + at) * Sh::TileT::kStride;
            i32x4 kf[2][kFrags];
#pragma unroll
            for (int c = 0; c < kFrags; ++c)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if constexpr (kStreamed) kf[u][c] = in.keys(now, at + 16 * u, c);
                    else kf[u][c] = Sh::keys(now, at + 16 * u, c);
                }
            keep_order();
            score([&](int u, int c) { return kf[u][c]; });
            ask(values, 0, vf[0]);
            keep_order();
            weigh(range[0], range[0].first_key(tile) + at);
            add(values);
            now = then;
            if constexpr (kStreamed) in.arrived();
            else if (tile + 1 < end) in.store(now);
            __syncthreads();
        }
    } else {
        char* const values = lds + wave * In::kTileBytes;
        for (; tile < end; tile += WAVES) {
            score([&](int u, int c) { return in.keys(u, c); });
            in.store_values(values);
            if (tile + WAVES < end) fetch(tile + WAVES, nullptr);
            lanes_exchange();
            ask(values, 0, vf[0]);
            if (kRanges == 2 && tile >= first_range) weigh(range[kRanges - 1], range[kRanges - 1].first_key(tile - first_range));
            else weigh(range[0], range[0].first_key(tile));
            add(values);
            lanes_exchange();
        }
    }

    // The waves' parts, brought to their common maximum and added in order.
    float mine_by[COLS];
#pragma unroll
    for (int n = 0; n < COLS; ++n) {
        l[n] = quads_sum(l[n]);
        if (l[n] == 0.f) m[n] = -kInf;
        if (quad == 0) {
            tops[key_wave * kRows + w0 + 16 * n + col] = m[n];
            totals[key_wave * kRows + w0 + 16 * n + col] = l[n];
        }
    }
    __syncthreads();  // also: the tiles' LDS is free
    float top[COLS], sum[COLS];
#pragma unroll
    for (int n = 0; n < COLS; ++n) {
        top[n] = tops[w0 + 16 * n + col];
#pragma unroll
        for (int x = 1; x < kKeyWaves; ++x) top[n] = fmaxf(top[n], tops[x * kRows + w0 + 16 * n + col]);
        const float less = top[n] == -kInf ? 0.f : top[n];
        sum[n] = 0.f;
#pragma unroll
        for (int x = 0; x < kKeyWaves; ++x)
            sum[n] += totals[x * kRows + w0 + 16 * n + col] * exp2_fast(tops[x * kRows + w0 + 16 * n + col] - less);
        mine_by[n] = exp2_fast(m[n] - less);
    }
    float* const sums = reinterpret_cast<float*>(lds);
    for (int x = 0; x < kKeyWaves; ++x) {
        if (x == key_wave) {
#pragma unroll
            for (int n = 0; n < COLS; ++n)
#pragma unroll
                for (int d = 0; d < kOut; ++d) {
                    f32x4* const at = reinterpret_cast<f32x4*>(sums + (w0 + 16 * n + col) * kSumStride + 16 * d + 4 * quad);
                    f32x4 y = x == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : *at;
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(o[d][n][e], mine_by[n], y[e]);
                    *at = y;
                }
        }
        __syncthreads();
    }
    if (quad == 0 && key_wave == 0) {
#pragma unroll
        for (int n = 0; n < COLS; ++n) {
            tops[w0 + 16 * n + col] = top[n];
            totals[w0 + 16 * n + col] = sum[n];
        }
    }
    __syncthreads();
    // Rows of the block, one a wave at a time: out, or the split's part of it.
    for (int row = wave; row < rows; row += WAVES) {
        float x0 = lane < a.D ? sums[row * kSumStride + lane] : 0.f;
        float x1 = lane + kWave < a.D ? sums[row * kSumStride + lane + kWave] : 0.f;
        float lm = tops[row], ll = totals[row];
        // A sum of weights that is NaN comes from a seen pair, and all of its row is NaN as it
        // lies, but where a bias of -inf masks that pair.
        const bool none = ll != ll;
        bool masks = false;
        if (none && biased) {
            const int column = heads < group ? row : row_of(r0 + row).h;
            for (int x = lane; x < a.bk.count; x += kWave) masks |= table[x * heads + column] == -kInf;
        }
        const bool n0 = none || !finite(x0), n1 = none || !finite(x1);
        if (ll == 0.f) {
            x0 = x1 = 0.f;
        } else if (none ? ballot(masks) != 0 : ballot(n0 || n1) != 0) {
            const Row at_row = row_of(r0 + row);
            const int column = heads < group ? row : at_row.h;
            CarefulKept<T, FORM> c(a, a.q.at<T>(at_row.b, g * group + at_row.h) + at_row.i * a.q.n);
            const int place = a.start.tokens + (kManySequences ? uniform(a.length(at_row.b)) : own_length) - a.Q + at_row.i;
            bool done = false;
#pragma unroll
            for (int x = 0; x < kRanges; ++x) {
                const Range<kTile, COLS>& at = range[x];
                const Seen sees = seen_of(a, place, at.base, at.limit);
                const int before = x == 0 ? 0 : first_range;
                for (int t = max(begin - before, 0); t < min(end - before, at.tiles) && !done; ++t)
                    for (int j = at.first_key(t); j < at.first_key(t) + kTile && !done; ++j)
                        if (sees(j)) {
                            const int64_t n = j;
                            c.add(at.k + n * at.kept->kn, at.v + n * at.kept->vn, at.k_scales + n * In::kScales,
                                  at.v_scales + n * In::kScales, biased ? bias_at(place - at.base - j, column) : 0.f);
                            done = none ? c.l != c.l : c.settled(n0, n1);
                        }
            }
            c.replace(none, n0, n1, x0, x1, lm, ll);
        }
        if (KIND == kBoth || part == nullptr) {
            const Row at_row = row_of(r0 + row);
            RowSum all{lm, ll, x0, x1};
            all.divide();
            all.write(out + ((static_cast<int64_t>(at_row.b) * a.Q + at_row.i) * a.H + g * group + at_row.h) * a.D, a.D);
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

// Parts: the start's blocks, then the caches', which fill the compute units beside and behind
// them (64 sequences of 512 tokens behind 16384, 32 heads over 8 of 128, bfloat16: 62 us, by two
// launches 73).  A start's block has 16 COLS rows of ROW_WAVES waves, a cache's 16 OWN_COLS.
// Registers: two waves a SIMD, one for 32-bit values, whose products take four times the operands.
template <typename T, int FORM, int DP, int COLS, int ROW_WAVES, int OWN_COLS>
__global__ __launch_bounds__(kStepThreads, FORM == kAny || (sizeof(T) == 4 && (FORM < kFour || COLS * OWN_COLS > 1)) ? 1 : 2) void attention_cache_kernel(
    const CacheArgs a, const CachePlan plan, T* __restrict__ out, float* __restrict__ parts, uint32_t first_block) {
    extern __shared__ __attribute__((aligned(16))) char cache_lds[];
    constexpr int kStartRows = 16 * COLS * ROW_WAVES, kOwnRows = 16 * OWN_COLS;
    // (A launch has fewer than 2^31 blocks; divisions of 64 bits are a hundred instructions each.)
    const uint32_t block = first_block + blockIdx.x, first = static_cast<uint32_t>(plan.start.units) * plan.start.splits;
    if (block < first) {
        // The row blocks of the same keys are eight blocks apart, on one XCD (whose L2 then
        // holds the keys for all of them).
        const uint32_t splits = plan.start.splits, all = a.G * splits, eights = 8u * plan.start.blocks;
        const uint32_t some = block / eights, left = min(8u, all - 8 * some), in = block - some * eights;
        const uint32_t row_block = in / left, keys = 8 * some + in - row_block * left, g = keys / splits, split_at = keys - g * splits;
        const int64_t place = (static_cast<int64_t>(g) * plan.start.blocks + row_block) * splits + split_at;
        attention_part<T, FORM, DP, COLS, ROW_WAVES, kStepWaves, kStart>(
            a, out, parts + place * plan.start.rows * part_width(DP), 0, static_cast<int>(g), static_cast<int>(row_block) * kStartRows,
            static_cast<int>(split_at), plan.start.splits, cache_lds);
    } else {
        const uint32_t at = block - first, unit = at / plan.own.splits, bg = unit / plan.own.blocks, b = bg / a.G;
        attention_part<T, FORM, DP, OWN_COLS, 1, kStepWaves, kOwn>(
            a, out, plan.joined ? parts + plan.start.floats + static_cast<int64_t>(at) * plan.own.rows * part_width(DP) : nullptr,
            static_cast<int>(b), static_cast<int>(bg - b * a.G), static_cast<int>(unit - bg * plan.own.blocks) * kOwnRows,
            static_cast<int>(at - unit * plan.own.splits), plan.own.splits, cache_lds);
    }
}

// Few keys: a sequence's rows with all that they see, the start's keys among them, in
// one block, without parts.  Eight waves, so that each has few tiles one after the other;
// four where the registers do not hold more.
constexpr int direct_waves(int size, int form, int DP) { return size == 4 && form < kFour && DP > 64 ? 4 : 8; }

template <typename T, int FORM, int DP>
__global__ __launch_bounds__(kWave * direct_waves(sizeof(T), FORM, DP), direct_waves(sizeof(T), FORM, DP) / 4) void attention_direct_kernel(
    const CacheArgs a, T* __restrict__ out, uint32_t first_block) {
    const uint32_t block = first_block + blockIdx.x;
    extern __shared__ __attribute__((aligned(16))) char cache_lds[];
    attention_part<T, FORM, DP, 1, 1, direct_waves(sizeof(T), FORM, DP), kBoth>(
        a, out, nullptr, static_cast<int>(block / a.G), static_cast<int>(block % a.G), 0, 0, 1, cache_lds);
}

// Kernels, by the rows of a start's block and of a cache's.
enum Shape { kDirect, kOne, kTwo, kPairs, kTwoTwo, kPairsTwo, kShapes };
struct ShapeRows {
    int cols, row_waves, own_cols;
    constexpr int start() const { return 16 * cols * row_waves; }
    constexpr int own() const { return 16 * own_cols; }
};
constexpr ShapeRows kShapeRows[kShapes] = {{1, 1, 1}, {1, 1, 1}, {2, 1, 1}, {2, 2, 1}, {2, 1, 2}, {2, 2, 2}};

template <typename T, int FORM>
hipError_t launch_cache_form(const CacheArgs& a, const CachePlan& plan, void* out, float* parts, hipStream_t stream) {
    return with_width(a.D, [&](auto width) {
        constexpr int DP = decltype(width)::value;
        auto launch = [&](auto* kernel, std::atomic<uint64_t>& allowed, int64_t blocks, int waves, size_t lds, auto... rest) {
            if (lds > kMostLds) return hipErrorInvalidValue;
            if (lds > kLdsFree) {
                const hipError_t err = allow_lds(kernel, allowed, kMostLds);
                if (err != hipSuccess) return err;
            }
            return in_launches(static_cast<uint32_t>(blocks), [&](uint32_t first, uint32_t count) {
                hipLaunchKernelGGL(kernel, dim3(count), dim3(kWave * waves), lds, stream, a, rest..., first);
            });
        };
        auto parted = [&](auto shape) {
            constexpr ShapeRows R = kShapeRows[decltype(shape)::value];
            using Start = StepLds<T, FORM, DP, R.cols, R.row_waves, kStepWaves>;
            using Own = StepLds<T, FORM, DP, R.own_cols, 1, kStepWaves>;
            const size_t own_lds = Own::kBytes + bias_lds(a, Own::kRows);
            static std::atomic<uint64_t> allowed;
            return launch(attention_cache_kernel<T, FORM, DP, R.cols, R.row_waves, R.own_cols>, allowed,
                          plan.start.units * plan.start.splits + plan.own.units * plan.own.splits, kStepWaves,
                          plan.start.units == 0 ? own_lds : std::max(Start::kBytes + bias_lds(a, Start::kRows), own_lds), plan,
                          static_cast<T*>(out), parts);
        };
        if constexpr (FORM == kAny) {  // (whose plans have no others)
            return parted(std::integral_constant<int, kTwoTwo>{});
        } else {
            switch (plan.shape) {
                case kDirect: {
                    constexpr int W = direct_waves(sizeof(T), FORM, DP);
                    using L = StepLds<T, FORM, DP, 1, 1, W>;
                    static std::atomic<uint64_t> allowed;
                    return launch(attention_direct_kernel<T, FORM, DP>, allowed, plan.own.units, W, L::kBytes + bias_lds(a, L::kRows),
                                  static_cast<T*>(out));
                }
                case kOne: return parted(std::integral_constant<int, kOne>{});
                case kTwo: return parted(std::integral_constant<int, kTwo>{});
                case kPairs: return parted(std::integral_constant<int, kPairs>{});
                case kPairsTwo: return parted(std::integral_constant<int, kPairsTwo>{});
                default: return parted(std::integral_constant<int, kTwoTwo>{});
            }
        }
    });
}

}  // namespace attn
}  // namespace pointops
