// Shared pieces of the attention kernels (gfx950): matrix-core fragments of
// the three types, tiles in LDS, which keys a query sees, and the bias by
// offset.
//
// Every product takes its tile operand (A, from LDS) by rows and its other
// operand (B) from registers, one column a lane: with keys as rows and queries
// as columns a lane holds the scores of one query, so that the softmax is a
// lane's own arithmetic, and the scores are, as they lie, the B operand of the
// next product.  What a lane holds of a 32 x 32 result is column lane % 32 and
// rows 8 g + 4 h + e (g, e = 0 .. 3, h = lane / 32) in register 4 g + e.
#pragma once

#include <atomic>
#include <type_traits>

#include "pointops_common.hpp"
#include "pointops_hip.h"

namespace pointops {
namespace attn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_inff();
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kOuter = 128;      // rows of a block that stay in registers, 32 a wave
constexpr int kMaxHead = 128;    // largest head width
constexpr int kMaxReach = 1024;  // the bias is constant beyond this offset

// A fragment is 16 bytes a lane: 8 values of 16 bits or 4 of 32.  As a row
// operand it holds bytes 32 c + 16 h .. + 15 of the lane's row (chunk c).
template <typename T>
constexpr int kPerFrag = 16 / static_cast<int>(sizeof(T));

// acc += A B over one chunk (16 values of 16 bits in one instruction, or 8
// of 32 bits in four; values 4 u + e of the two half-waves meet in step e).
template <typename T>
__device__ __forceinline__ f32x16 mma(i32x4 a, i32x4 b, f32x16 acc) {
    if constexpr (sizeof(T) == 4) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], acc, 0, 0, 0);
        return acc;
    } else if constexpr (__is_same(T, bf16)) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
    }
}

// Registers p[0 .. kPerFrag - 1] of a result as a B fragment of T (rounded to
// nearest even for the 16-bit types).
template <typename T>
__device__ __forceinline__ i32x4 as_fragment(const float* p) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(i32x4, f32x4{p[0], p[1], p[2], p[3]});
    } else if constexpr (__is_same(T, bf16)) {
        bf16x8 r;
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = static_cast<bf16>(p[e]);
        return __builtin_bit_cast(i32x4, r);
    } else {
        f16x8 r;
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = static_cast<f16>(p[e]);
        return __builtin_bit_cast(i32x4, r);
    }
}

template <typename T>
__device__ __forceinline__ float to_float(T v) { return static_cast<float>(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v) { return static_cast<T>(v); }

// Element e of a fragment.
template <typename T>
__device__ __forceinline__ float element(i32x4 f, int e) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(f32x4, f)[e];
    else if constexpr (__is_same(T, bf16)) return static_cast<float>(__builtin_bit_cast(bf16x8, f)[e]);
    else return static_cast<float>(__builtin_bit_cast(f16x8, f)[e]);
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The sum and the maximum of a value over the two half-waves.
__device__ __forceinline__ float halves_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(f2i(v), f2i(v), false, false);
    return i2f(r[0]) + i2f(r[1]);
}
__device__ __forceinline__ float halves_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(f2i(v), f2i(v), false, false);
    return fmaxf(i2f(r[0]), i2f(r[1]));
}

// The sum over aligned groups of L lanes, in every lane.
template <int L>
__device__ __forceinline__ float group_sum(float v) {
    if constexpr (L >= 2) v += i2f(dpp<kDppQuadXor1>(f2i(v)));
    if constexpr (L >= 4) v += i2f(dpp<kDppQuadXor2>(f2i(v)));
    if constexpr (L >= 8) v += i2f(dpp<kDppRowHalfMirror>(f2i(v)));
    if constexpr (L >= 16) v += i2f(dpp<kDppRowMirror>(f2i(v)));
    if constexpr (L >= 32) v += __shfl_xor(v, 16);
    if constexpr (L >= 64) v += __shfl_xor(v, 32);
    return v;
}

__device__ __forceinline__ float wave_sum(float v) { return group_sum<kWave>(v); }

// ------------------------------------------------------------------ tiles
constexpr int kRawBuffer = 0x00027000;  // word 3 of a buffer descriptor for plain bytes

// 16 bytes of a row of `width` elements from element `at` on, zeros behind its
// end.  VEC: rows are 16-byte aligned and `width` is a multiple of kPerFrag.  Others
// are read value by value, their kernels serve calls with and without a bias and do not
// split rows between waves (4 x 2048, 8 heads over 2 of 64, window 512: bfloat16 65 us
// forward and 260 with gradients, aligned 25 and 134; float32 122 and 563, 102 and 444).
template <typename T, bool VEC>
__device__ __forceinline__ i32x4 load_row(const T* row, int at, int width) {
    i32x4 r = {0, 0, 0, 0};
    if constexpr (VEC) {
        if (at < width) r = *reinterpret_cast<const i32x4*>(row + at);
    } else {
        union { i32x4 v; T e[kPerFrag<T>]; } u;
        u.v = r;
#pragma unroll
        for (int e = 0; e < kPerFrag<T>; ++e)
            if (at + e < width) u.e[e] = row[at + e];
        r = u.v;
    }
    return r;
}

// Rows of DP elements in LDS, an odd number of 16-byte units apart: the row
// operands' reads of 16 rows fall on all banks.  Rows of 256 bytes are 3 units
// longer, as with one the transposing reads of four neighbouring rows would
// meet in the same banks.
template <typename T, int DP>
struct Tile {
    static constexpr int kBytes = DP * static_cast<int>(sizeof(T));
    static constexpr int kStride = kBytes + (kBytes == 256 ? 48 : 16);
    static constexpr int kChunks = DP * static_cast<int>(sizeof(T)) / 32;  // of a row operand
    static constexpr int kRowsPerFrag = 2 * kPerFrag<T>;  // rows that a transposed fragment spans

    // Row operand: row `row0` + lane % 32, chunk c.
    __device__ static __forceinline__ i32x4 rows(const char* tile, int row0, int c) {
        const int lane = lane_id();
        return *reinterpret_cast<const i32x4*>(tile + (row0 + lane % 32) * kStride + 32 * c + 16 * (lane / 32));
    }

    // Transposed operand: its row is column d0 + lane % 32 of the tile, its
    // values the tile's rows row0 + 8 g + 4 h + e in the order of a result's
    // registers.  16-bit types by the transposing read (16 lanes take a 4 x 16
    // block, each one column), 32-bit ones value by value.
    __device__ static __forceinline__ i32x4 columns(const char* tile, int row0, int d0) {
        const int lane = lane_id(), h = lane / 32;
        if constexpr (sizeof(T) == 4) {
            const char* p = tile + (row0 + 4 * h) * kStride + 4 * (d0 + lane % 32);
            i32x4 r;
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = *reinterpret_cast<const int*>(p + e * kStride);
            return r;
        } else {
            const int i = lane % 16;
            const char* p = tile + (row0 + 4 * h + i / 4) * kStride + 2 * (d0 + 16 * ((lane / 16) % 2) + 4 * (i % 4));
            typedef __attribute__((address_space(3))) s16x4 lds4;
            const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p));
            const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 8 * kStride));
            const i32x2 a = __builtin_bit_cast(i32x2, x), b = __builtin_bit_cast(i32x2, y);
            return i32x4{a[0], a[1], b[0], b[1]};
        }
    }
};

// The compiler's scheduler keeps what is before this before what is behind it.
// The products below ask for their operands as a batch, a phase ahead of their
// use: left to itself it reads each right before its product, which then waits
// for LDS (at one wave a SIMD that was two thirds of the time).
__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0); }

// Between a wave's stores to LDS and its other lanes' reads of them (or the next
// stores): the hardware keeps a wave's LDS accesses in order, and neither the compiler's
// memory passes nor its scheduler may change it.  No instruction.
__device__ __forceinline__ void lanes_exchange() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Row operands of a tile's rows row0 .. row0 + 31, all chunks.
template <typename T, int DP>
struct RowFrags {
    static constexpr int kChunks = Tile<T, DP>::kChunks;
    i32x4 f[kChunks];
    __device__ __forceinline__ void load(const char* tile, int row0) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) f[c] = Tile<T, DP>::rows(tile, row0, c);
    }
    __device__ __forceinline__ f32x16 times(const i32x4 (&b)[kChunks]) const {
        f32x16 acc = {};
#pragma unroll
        for (int c = 0; c < kChunks; ++c) acc = mma<T>(f[c], b[c], acc);
        return acc;
    }
};

// Transposed operands of all columns, of the rows that one fragment spans.
template <typename T, int DP>
struct ColumnFrags {
    i32x4 f[DP / 32];
    __device__ __forceinline__ void load(const char* tile, int row0) {
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) f[d] = Tile<T, DP>::columns(tile, row0, 32 * d);
    }
    __device__ __forceinline__ void add(i32x4 b, f32x16 (&acc)[DP / 32]) const {
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[d] = mma<T>(f[d], b, acc[d]);
    }
};

// A tile's way from memory to LDS through a block's registers: requested
// before the one ahead of it is used.  Rows outside [first, high) and columns
// behind the row's width are zeros: where rows allow 16-byte reads, by a buffer
// descriptor that ends with the last row (a read behind its end returns zeros
// and touches nothing), so that a thread's offsets are the same for all tiles.
template <typename T, int DP, int ROWS, bool VEC>
struct Stage {
    static constexpr int kPerRow = DP * static_cast<int>(sizeof(T)) / 16;
    static constexpr int kPieces = ROWS * kPerRow / kThreads;
    static_assert(ROWS * kPerRow % kThreads == 0);
    i32x4 r[kPieces];

    // Rows first .. first + ROWS - 1 of [0, high); all arguments are uniform.
    __device__ __forceinline__ void load(const T* base, int64_t stride, int first, int high, int width) {
        if constexpr (VEC) {
            const int64_t bytes = (static_cast<int64_t>(high - 1 - first) * stride + width) * static_cast<int64_t>(sizeof(T));
            const auto rows = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<T*>(base + first * stride), 0,
                first < high ? static_cast<int>(min(bytes, int64_t(INT32_MAX))) : 0, kRawBuffer);
            const uint32_t step = static_cast<uint32_t>(stride) * sizeof(T);
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const uint32_t at = i * kThreads + threadIdx.x, col = at % kPerRow;
                const uint32_t offset = static_cast<int>(col) * kPerFrag<T> < width ? at / kPerRow * step + col * 16 : 0x80000000u;
                r[i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rows, offset, 0, 0));
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int at = i * kThreads + static_cast<int>(threadIdx.x);
                const int row = first + at / kPerRow;
                r[i] = i32x4{0, 0, 0, 0};
                if (row < high) r[i] = load_row<T, false>(base + row * stride, at % kPerRow * kPerFrag<T>, width);
            }
        }
    }
    // Rows times by(row), row 0 being `first`.  Seldom called: what follows from the
    // thread's number is worked out here, not kept in registers through a kernel's loop.
    template <typename F>
    __device__ __forceinline__ void scale(F by) {
        int thread = threadIdx.x;
        asm volatile("" : "+v"(thread));
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const float f = by((i * kThreads + thread) / kPerRow);
            float x[kPerFrag<T>];
#pragma unroll
            for (int e = 0; e < kPerFrag<T>; ++e) x[e] = element<T>(r[i], e) * f;
            r[i] = as_fragment<T>(x);
        }
    }
    __device__ __forceinline__ void store(char* tile) const {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int at = i * kThreads + static_cast<int>(threadIdx.x);
            *reinterpret_cast<i32x4*>(tile + at / kPerRow * Tile<T, DP>::kStride + at % kPerRow * 16) = r[i];
        }
    }
};

// The running maximum may lie this far (in units of log 2) below the true one:
// weights up to 2^8 cost no precision, and outputs are rescaled seldom.
constexpr float kSlack = 8.f;

// Rows of an inner tile: 64, or 32 where a value has 32 bits (the same LDS).
template <typename T>
constexpr int kInner = sizeof(T) == 4 ? 32 : 64;

// Where 128 rows a block would leave compute units with one block or none, a
// block takes 64: two waves share each 32 of them and take half of every inner
// tile (of 64 rows) each, and their sums are joined in LDS at the end.
template <typename T, int SPLIT>
struct Cut {
    static constexpr int kRows = kOuter / SPLIT;  // of a block
    static constexpr int kInnerRows = SPLIT == 2 ? 64 : kInner<T>;
    static constexpr int kSub = kInnerRows / 32 / SPLIT;  // 32-row pieces of an inner tile that a wave takes
};
inline bool few_blocks(int64_t blocks) { return blocks < 512; }
// Rows of up to 256 bytes: the wider ones' tiles of 64 would leave no LDS for a bias.
template <typename T, int DP>
constexpr bool kSplits = DP * sizeof(T) <= 256;

// A wave's registers to its partner, lane by lane.
template <int N>
__device__ __forceinline__ void put_sums(float* lds, const f32x16 (&v)[N]) {
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) lds[(d * 16 + r) * kWave + lane_id()] = v[d][r];
}
template <int N>
__device__ __forceinline__ void get_sums(const float* lds, f32x16 (&v)[N], float keep, float by) {
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) v[d][r] = __builtin_fmaf(lds[(d * 16 + r) * kWave + lane_id()], by, v[d][r] * keep);
}

// Registers from .. from + 3 of a result to elements at .. at + 3 of a row
// (VEC: the row's width is a multiple of 4 and its start aligned to as many).
template <typename T, bool VEC>
__device__ __forceinline__ void store4(T* row, int at, int width, const f32x16& v, int from) {
    T piece[4];
#pragma unroll
    for (int f = 0; f < 4; ++f) piece[f] = from_float<T>(v[from + f]);
    if constexpr (VEC) {
        if (at < width) __builtin_memcpy(__builtin_assume_aligned(row + at, 4 * sizeof(T)), piece, sizeof piece);
    } else {
#pragma unroll
        for (int f = 0; f < 4; ++f)
            if (at + f < width) row[at + f] = piece[f];
    }
}

// -------------------------------------------------------------- arguments
struct Rows {
    const void* p;
    int64_t b, n, h;  // strides of batch, token and head, in elements
    template <typename T>
    __device__ __forceinline__ const T* at(int64_t batch, int64_t head) const {
        return static_cast<const T*>(p) + batch * b + head * h;
    }
};

// Buckets of an offset: edge[0 .. n - 1] ascending; count = n + 1, or twice
// that where later keys have buckets of their own.
struct Buckets {
    int n, count;
    int edge[255];
};

struct Args {
    Rows q, k, v;
    const void* bias;  // (bk.count, H), or null
    const void* lengths;
    int B, Q, N, H, G, D;
    int window, sinks;  // window in [1, N + 1]
    int reach;          // the last edge: the bias is constant from there on
    int length_bits;
    bool causal;
    float scale_log2;  // scale log2(e): scores are in units of log 2
    float scale;
    Buckets bk;

    // Uniform, as b is.
    __device__ __forceinline__ int length(int b) const {
        if (lengths == nullptr) return N;
        const int64_t l = length_bits == 64 ? static_cast<const int64_t*>(lengths)[b]
                                            : static_cast<const int32_t*>(lengths)[b];
        return uniform(static_cast<int>(l < 0 ? 0 : l > N ? N : l));
    }
};

// Keys that the query at position p sees: low .. low + count - 1, and those
// below `first`.
struct Seen {
    int low, count, first;
    __device__ __forceinline__ bool operator()(int j) const {
        return static_cast<uint32_t>(j - low) < static_cast<uint32_t>(count) || j < first;
    }
};

__device__ __forceinline__ int seen_low(const Args& a, int p) { return max(0, p - a.window + 1); }
__device__ __forceinline__ int seen_high(const Args& a, int p, int len) {
    return a.causal ? p : min(len - 1, p + a.window - 1);
}
__device__ __forceinline__ int seen_first(const Args& a, int p, int len) {
    return min(a.sinks, a.causal ? min(p + 1, len) : len);
}
__device__ __forceinline__ Seen seen_by(const Args& a, int p, int len) {
    if (p < 0 || p >= len) return {0, 0, 0};
    const int low = seen_low(a, p);
    return {low, seen_high(a, p, len) - low + 1, seen_first(a, p, len)};
}

// The tiles of `inner` keys that a block of rows sees: 0 .. first_end - 1 (the
// first keys'), then low .. end - 1 (the window's).
struct Walk {
    int first_end = 0, low = 0, end = 0;
    __device__ __forceinline__ Walk(const Args& a, int p_first, int p_last, int len, int inner) {
        if (p_first > p_last) return;
        first_end = (seen_first(a, p_last, len) + inner - 1) / inner;
        low = max(first_end, seen_low(a, p_first) / inner);
        end = max(first_end, seen_high(a, p_last, len) / inner + 1);
    }
    __device__ __forceinline__ int begin() const { return first_end > 0 ? 0 : low; }
    __device__ __forceinline__ int after(int t) const { return t + 1 >= first_end && t + 1 < low ? low : t + 1; }
};

// A block's place among `outer` heads (or key heads) of `inner` blocks each.
// The hardware deals blocks to the 8 XCDs in turn: where the heads are a
// multiple of 8, each XCD takes an eighth of them (whose keys and values then
// share its L2), their first blocks before their second ones.
struct Place {
    int outer, inner;
};
__device__ __forceinline__ Place place(int outer, int inner) {
    const uint32_t id = blockIdx.x, n = static_cast<uint32_t>(outer);
    if (n % 8 != 0) return {static_cast<int>(id % n), static_cast<int>(id / n)};
    const uint32_t xcd = id % 8, rank = id / 8, each = n / 8;
    return {static_cast<int>(xcd * each + rank % each), static_cast<int>(rank / each)};
}

// Block `rank` of a head's `blocks`, in the order in which they are handed out:
// the later half from the last one down, then the earlier half from the first
// one up.  A causal call's rows grow with their position, and blocks that meet
// on a compute unit are then a long and a short one.
__device__ __forceinline__ int folded(int rank, int blocks) {
    const int late = (blocks + 1) / 2;
    return rank < late ? blocks - 1 - rank : rank - late;
}

// ------------------------------------------------------------------- bias
// A block's bias by offset (query's position less key's) in LDS, in units of
// log 2: entry offset + reach + kMargin, the ends repeated over the margins,
// so that a tile with any offset inside the reach indexes it without a clamp.
constexpr int kMargin = kOuter + 64;
__host__ __device__ inline int bias_entries(int reach) { return 2 * (reach + kMargin) + 1; }

// Bucket of an offset: the number of edges at or below its distance; the
// buckets of later keys, where there are any, follow those of earlier ones.
__device__ __forceinline__ int bucket_of(const Buckets& bk, const int* edges, int offset) {
    const bool later = offset < 0;
    const bool two_sided = bk.count > bk.n + 1;
    const int d = later ? (two_sided ? -offset : 0) : offset;
    int low = 0, high = bk.n;  // edges below `low` are <= d, those from `high` on are not
    while (low < high) {
        const int mid = (low + high) >> 1;
        if (edges[mid] <= d) low = mid + 1;
        else high = mid;
    }
    return low + (later && two_sided ? bk.n + 1 : 0);
}

// v log2(e), kept finite where v is: a mask of the type's lowest value stays
// one that all keys of a row can share.
__device__ __forceinline__ float bias_log2(float v) {
    const float w = v * kLog2e;
    if (w - w != 0.f && v - v == 0.f) return v < 0.f ? -3e38f : 3e38f;
    return w;
}

// One offset's bias for the whole wave, without a table.
template <typename T>
__device__ __forceinline__ float one_bias(const Args& a, int head, int offset) {
    if (a.bias == nullptr) return 0.f;
    return bias_log2(to_float(static_cast<const T*>(a.bias)[static_cast<int64_t>(bucket_of(a.bk, a.bk.edge, offset)) * a.H + head]));
}

// Fills the table for head `head` (edges: LDS, bk.n ints).  The caller's
// next barrier makes it visible; this one has a barrier of its own.
template <typename T>
__device__ __forceinline__ void fill_bias(const Args& a, int head, float* table, int* edges) {
    for (int i = threadIdx.x; i < a.bk.n; i += kThreads) edges[i] = a.bk.edge[i];
    __syncthreads();
    const T* bias = static_cast<const T*>(a.bias) + head;
    for (int i = threadIdx.x; i < bias_entries(a.reach); i += kThreads) {
        const int b = bucket_of(a.bk, edges, i - a.reach - kMargin);
        table[i] = bias_log2(to_float(bias[static_cast<int64_t>(b) * a.H]));
    }
}

// ------------------------------------------------------------ careful rows
// Only what came out of the products not finite is formed again: finite values have
// met no infinity or NaN.  And only until it is not finite again, which is then its
// own: what a place that is no number in a seen pair costs ends there, and a pass
// over all pairs is left to values that are finite without their masked neighbours.
__device__ __forceinline__ bool finite(float x) { return x - x == 0.f; }

// A lane's values of a result that are not finite: bit 16 d + register.
template <int N>
__device__ __forceinline__ uint64_t odd_values(const f32x16 (&v)[N]) {
    uint64_t odd = 0;
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) odd |= finite(v[d][r]) ? 0 : uint64_t(1) << (16 * d + r);
    return odd;
}
// Whether value `c` of the result's row (lane column) r is one of them, r uniform.
__device__ __forceinline__ bool odd_value(uint64_t odd, int r, int c) {
    const int low = static_cast<int>(odd), high = static_cast<int>(odd >> 32);
    const uint64_t of[2] = {static_cast<uint32_t>(readlane(low, r)) | uint64_t(static_cast<uint32_t>(readlane(high, r))) << 32,
                            static_cast<uint32_t>(readlane(low, r + 32)) | uint64_t(static_cast<uint32_t>(readlane(high, r + 32))) << 32};
    const uint64_t mine = (c & 4) != 0 ? of[1] : of[0];
    return (mine >> (c / 32 * 16 + c % 32 / 8 * 4 + c % 4) & 1) != 0;
}

// One query by a whole wave, key by key, for rows whose result is not finite:
// there a product with a masked key's infinity or NaN may have spread.  Only
// keys that the row sees are added (one whose score is -inf, or whose bias is,
// whatever it holds, has no weight and is left out).  Lane l holds elements l and
// l + 64, of which it needs those that came out not finite (n0, n1).
template <typename T>
struct CarefulRow {
    const Args& a;
    const T *k, *v;
    float q0, q1, m = -kInf, l = 0.f, o0 = 0.f, o1 = 0.f;
    bool d0, d1;

    __device__ __forceinline__ CarefulRow(const Args& args, int b, int g, const T* q) : a(args) {
        const int lane = lane_id();
        k = a.k.at<T>(b, g) + lane;
        v = a.v.at<T>(b, g) + lane;
        d0 = lane < a.D;
        d1 = lane + kWave < a.D;
        q0 = d0 ? to_float(q[lane]) : 0.f;
        q1 = d1 ? to_float(q[lane + kWave]) : 0.f;
    }
    __device__ __forceinline__ void add(int64_t j, float bias) {
        if (bias == -kInf) return;
        const float k0 = d0 ? to_float(k[j * a.k.n]) : 0.f, k1 = d1 ? to_float(k[j * a.k.n + kWave]) : 0.f;
        const float s = wave_sum((d0 ? q0 * k0 : 0.f) + (d1 ? q1 * k1 : 0.f)) * a.scale_log2 + bias;
        if (s == -kInf) return;
        const float top = fmaxf(m, s), keep = m == -kInf ? 0.f : exp2_fast(m - top), w = exp2_fast(s - top);
        m = top;
        l = l * keep + w;
        o0 = o0 * keep + (d0 ? w * to_float(v[j * a.v.n]) : 0.f);
        o1 = o1 * keep + (d1 ? w * to_float(v[j * a.v.n + kWave]) : 0.f);
    }
    // Whether all that is needed has come out not finite again.
    __device__ __forceinline__ bool settled(bool n0, bool n1) const {
        return ballot((n0 && finite(o0)) || (n1 && finite(o1))) == 0;
    }
};

// The same for gradients: one query and one key at a time, of which a wave holds
// elements l and l + 64 in lane l.
template <typename T>
struct CarefulPair {
    float x0 = 0.f, x1 = 0.f;
    __device__ __forceinline__ void load(const T* row, int width) {
        const int lane = lane_id();
        x0 = lane < width ? to_float(row[lane]) : 0.f;
        x1 = lane + kWave < width ? to_float(row[lane + kWave]) : 0.f;
    }
    __device__ __forceinline__ float dot(const CarefulPair& y) const { return wave_sum(x0 * y.x0 + x1 * y.x1); }
    __device__ __forceinline__ void add(float w, const CarefulPair& y) {
        x0 = __builtin_fmaf(w, y.x0, x0);
        x1 = __builtin_fmaf(w, y.x1, x1);
    }
};

// ---------------------------------------------------------------- dispatch
// Head widths are padded to a multiple of 32.
template <typename F>
hipError_t with_width(int64_t D, F f) {
    if (D <= 32) return f(std::integral_constant<int, 32>{});
    if (D <= 64) return f(std::integral_constant<int, 64>{});
    if (D <= 96) return f(std::integral_constant<int, 96>{});
    return f(std::integral_constant<int, 128>{});
}

// Whether 16-byte reads through a buffer descriptor serve these rows: aligned,
// one behind the other, and a tile of them within 2 GiB.
template <typename T>
bool vector_rows(const Rows& r, int64_t D) {
    const int64_t n = kPerFrag<T>;
    return r.n >= D && r.n < (int64_t(1) << 22) && reinterpret_cast<uintptr_t>(r.p) % 16 == 0 && r.b % n == 0 && r.n % n == 0 && r.h % n == 0 && D % n == 0;
}

// Allows a kernel `most` bytes of dynamic LDS, once per device (the limit belongs
// to the process: each kernel asks for the most that any call of it needs).
template <typename K>
inline hipError_t allow_lds(K kernel, std::atomic<uint64_t>& allowed, size_t most) {
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

// relative_bias.hip: reads the host's edges; false if they are none.
bool read_buckets(const int32_t* edges, int n, int count, int64_t most, Buckets* out);

// Adds a block's sums by offset (LDS, `entries` of them, offset o at entry o +
// zero; the outermost buckets of a side take what lies beyond) by buckets:
// dst[0 .. count - 1].  edge: bk.edge, or a copy of it.  Eight lanes a bucket.
__device__ __forceinline__ void add_buckets(const Buckets& bk, const int* edge, const float* sums, int entries, int zero,
                                            float* dst) {
    const int side = bk.n + 1;
    const bool two_sided = bk.count > side;
    for (int first = 0; first < bk.count; first += kThreads / 8) {
        const int bucket = first + static_cast<int>(threadIdx.x) / 8, e = bucket % side;
        float all = 0.f;
        if (bucket < bk.count) {
            const int d_low = e == 0 ? 0 : edge[e - 1], d_high = e == bk.n ? INT32_MAX : edge[e] - 1;
            int64_t low = static_cast<int64_t>(zero) + d_low, high = static_cast<int64_t>(zero) + d_high;
            if (bucket >= side) {
                low = static_cast<int64_t>(zero) - d_high;
                high = static_cast<int64_t>(zero) - max(d_low, 1);
            } else if (e == 0 && !two_sided) {
                low = 0;  // later keys have no buckets of their own
            }
            const int from = static_cast<int>(max(low, int64_t(0))), to = static_cast<int>(min(high, int64_t(entries - 1)));
#pragma unroll 4
            for (int i = from + static_cast<int>(threadIdx.x) % 8; i <= to; i += 8) all += sums[i];
        }
        all = group_sum<8>(all);
        if (bucket < bk.count && threadIdx.x % 8 == 0) dst[bucket] = all;
    }
}

// relative_bias.hip: grad[bucket][h] (of type POINTOPS_*) from part (B, H,
// blocks, count).  Given the bias itself (of the same type), entries of -inf have
// gradients of zero, whatever masked places have left in their sums.
hipError_t join_buckets(const float* part, int B, int H, int64_t blocks, int count, int type, const void* bias, void* grad,
                        hipStream_t stream);

// The device arguments of a call, and whether it is one that the kernels take.
bool read_args(const pointops_attention* in, Args* out);

}  // namespace attn
}  // namespace pointops
