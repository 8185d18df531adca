// A cache in 8 or 4 bits: writing new tokens to it and reading it back.
//
// Both are bound by memory: 8 x 16384 tokens of 8 heads of 128, float16 to 8 bits and back, take 169
// and 158 us, 4.8 and 5.1 TB/s of what they read and write (a large copy: 4.7).  Four
// neighbouring lanes hold a group of 32 values, eight each (16 bytes of a 16-bit type),
// and find its scale among themselves; neighbouring lanes are pieces of a row, then the
// tokens behind it, so that codes are written and read in whole lines (rows of 64 bytes
// for 4 bits and 128 values).
#include <algorithm>

#include "quantized_cache.hpp"

namespace pointops {
namespace attn {
namespace {

// One side (keys, values) of the cache and of the tokens.
struct Side {
    const void* rows;   // of the tokens, strides in elements
    int64_t b, n, h;
    uint8_t *codes, *scales;
};

struct CacheCall {
    Side side[2];
    const void *lengths, *starts;
    int length_bits, start_bits;
    int64_t cache_b, cache_h;  // strides of the cache, in rows
    int B, G, D, N, T;         // T: tokens of the call
    int at_once;               // values of a row's pieces that are read or written at once: 8, 4 or 1
};

__device__ __forceinline__ int64_t value_at(const void* p, int bits, int b) {
    return bits == 64 ? static_cast<const int64_t*>(p)[b] : static_cast<const int32_t*>(p)[b];
}

// Lanes of a row of D values, eight each, a whole number of groups.
__host__ __device__ constexpr int lanes_of(int D) { return padded(D) / 8; }

struct Piece {
    int side, b, g, t, at;  // at: the first of its eight values
    bool any;
};

// A block's pieces: whole rows of one key head's tokens (of 96 values 21, four threads
// are left over), so that no thread divides by more than a row's lanes.
__host__ __device__ constexpr int rows_of(int D) { return kThreads / lanes_of(D); }
__device__ __forceinline__ Piece piece_of(const CacheCall& c, int tokens, uint32_t blocks, uint32_t first) {
    const uint32_t block = first + blockIdx.x, chunk = block % blocks, unit = block / blocks, lanes = lanes_of(c.D);
    const uint32_t row = threadIdx.x * (65536 / lanes + 1) >> 16;  // of fewer than 256 threads, exactly
    Piece p;
    p.t = static_cast<int>(chunk * rows_of(c.D) + row);
    p.at = static_cast<int>(threadIdx.x - row * lanes) * 8;
    p.any = static_cast<int>(row) < rows_of(c.D) && p.t < tokens;
    p.side = static_cast<int>(unit % 2);
    p.g = static_cast<int>(unit / 2 % c.G);
    p.b = static_cast<int>(unit / 2 / c.G);
    return p;
}

// N values, at a multiple of 16 bytes or of their size if they are fewer.  What is read back is
// written past the caches (4 x 8192 tokens, 8 heads of 128, 4 bits, with a write of 2048: 58 us
// through them, 37 past them; what is read gains nothing by it).
template <typename T, int N>
struct Words {
    static constexpr int kBytes = N * static_cast<int>(sizeof(T));
    using Word = std::conditional_t<kBytes % 16 == 0, i32x4, i32x2>;
    static constexpr int kCount = kBytes / static_cast<int>(sizeof(Word));
    union {
        Word w[kCount];
        T v[N];
    };
};
template <typename T, int N>
__device__ __forceinline__ void get(const T* from, float* x) {
    Words<T, N> words;
#pragma unroll
    for (int i = 0; i < Words<T, N>::kCount; ++i) {
        const auto* const at = reinterpret_cast<const typename Words<T, N>::Word*>(from) + i;
        words.w[i] = *at;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = to_float(words.v[e]);
}
template <typename T, int N>
__device__ __forceinline__ void put(T* to, const T* x) {
    Words<T, N> words;
#pragma unroll
    for (int e = 0; e < N; ++e) words.v[e] = x[e];
#pragma unroll
    for (int i = 0; i < Words<T, N>::kCount; ++i) {
        auto* const at = reinterpret_cast<typename Words<T, N>::Word*>(to) + i;
        __builtin_nontemporal_store(words.w[i], at);
    }
}

template <typename T, int BITS>
__global__ __launch_bounds__(kThreads) void cache_write_kernel(const CacheCall c, uint32_t blocks, uint32_t first) {
    const Piece p = piece_of(c, c.T, blocks, first);
    const Side& s = c.side[p.side];
    int64_t length = c.N;
    if (c.lengths != nullptr) length = min(max(value_at(c.lengths, c.length_bits, p.b), int64_t(0)), int64_t(c.N));
    // (A start that far off leaves nothing to write, and none of its sums passes 64 bits.)
    int64_t start = length - c.T;
    if (c.starts != nullptr) start = min(max(value_at(c.starts, c.start_bits, p.b), -int64_t(c.T)), int64_t(c.N));
    const int64_t place = start + p.t;
    const bool here = p.any && place >= 0 && place < length;  // of a row's lanes all or none

    float x[8];
    const T* const row = static_cast<const T*>(s.rows) + p.b * s.b + p.t * s.n + p.g * s.h;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
    if (here) {
        if (c.at_once == 8) {
            if (p.at < c.D) get<T, 8>(row + p.at, x);
        } else if (c.at_once == 4) {
            if (p.at < c.D) get<T, 4>(row + p.at, x);
            if (p.at + 4 < c.D) get<T, 4>(row + p.at + 4, x + 4);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (p.at + e < c.D) x[e] = to_float(row[p.at + e]);
        }
    }
    // As whole numbers, magnitudes are in their order, infinity and NaN above all.
    int most = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, f2i(x[e]) & 0x7fffffff);
    most = max(most, dpp<kDppQuadXor1>(most));
    most = max(most, dpp<kDppQuadXor2>(most));
    if (!here) return;
    const uint32_t byte = scale_byte<BITS>(i2f(most));
    // The codes of a group that is no number are zeros: its scale says so.
    const float scale = scale_of(byte);
    const int64_t at = p.b * c.cache_b + p.g * c.cache_h + place;
    if constexpr (BITS == 8) {
        s16x2 low = {0, 0}, high = {0, 0};
        if (byte != kNoNumber) {
            low = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(low, x[0], x[1], scale, false);
            low = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(low, x[2], x[3], scale, true);
            high = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(high, x[4], x[5], scale, false);
            high = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(high, x[6], x[7], scale, true);
        }
        *reinterpret_cast<i32x2*>(s.codes + at * padded(c.D) + p.at) =
            i32x2{__builtin_bit_cast(int, low), __builtin_bit_cast(int, high)};
    } else {
        uint32_t codes = 0;
        if (byte != kNoNumber) {
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], scale, 0);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], scale, 1);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], scale, 2);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], scale, 3);
        }
        *reinterpret_cast<uint32_t*>(s.codes + at * (padded(c.D) / 2) + p.at / 2) = codes;
    }
    if (p.at % kGroup == 0) s.scales[at * (padded(c.D) / kGroup) + p.at / kGroup] = static_cast<uint8_t>(byte);
}

template <typename T, int BITS>
__global__ __launch_bounds__(kThreads) void cache_read_kernel(const CacheCall c, T* __restrict__ k, T* __restrict__ v,
                                                              uint32_t blocks, uint32_t first) {
    const Piece p = piece_of(c, c.N, blocks, first);
    if (!p.any || p.at >= c.D) return;
    const Side& s = c.side[p.side];
    const int64_t at = p.b * c.cache_b + p.g * c.cache_h + p.t;
    const float scale = scale_of(s.scales[at * (padded(c.D) / kGroup) + p.at / kGroup]);
    f32x2 x[4];
    if constexpr (BITS == 8) {
        const i32x2 codes = *reinterpret_cast<const i32x2*>(s.codes + at * padded(c.D) + p.at);
        x[0] = decode<8, 0>(codes[0], scale);
        x[1] = decode<8, 1>(codes[0], scale);
        x[2] = decode<8, 0>(codes[1], scale);
        x[3] = decode<8, 1>(codes[1], scale);
    } else {
        const uint32_t codes = *reinterpret_cast<const uint32_t*>(s.codes + at * (padded(c.D) / 2) + p.at / 2);
        x[0] = decode<4, 0>(codes, scale);
        x[1] = decode<4, 1>(codes, scale);
        x[2] = decode<4, 2>(codes, scale);
        x[3] = decode<4, 3>(codes, scale);
    }
    T piece[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) piece[e] = from_float<T>(x[e / 2][e % 2]);
    T* const row = (p.side == 0 ? k : v) + ((static_cast<int64_t>(p.b) * c.N + p.t) * c.G + p.g) * c.D + p.at;
    if (c.at_once == 8) {
        put<T, 8>(row, piece);
    } else if (c.at_once == 4) {
        put<T, 4>(row, piece);
        if (p.at + 4 < c.D) put<T, 4>(row + 4, piece + 4);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (p.at + e < c.D) row[e] = piece[e];
    }
}

bool read_cache(const pointops_cache* in, CacheCall* c) {
    const int64_t limit = (int64_t(1) << 30) - 1024;
    if (in == nullptr || in->B < 0 || in->N < 0 || in->G < 0 || in->D < 1 || in->D > kMaxHead) return false;
    if (in->B > limit || in->N > limit || in->G > limit || (in->bits != 8 && in->bits != 4)) return false;
    c->side[0] = {nullptr, 0, 0, 0, static_cast<uint8_t*>(in->k), in->k_scales};
    c->side[1] = {nullptr, 0, 0, 0, static_cast<uint8_t*>(in->v), in->v_scales};
    c->lengths = c->starts = nullptr;
    c->length_bits = c->start_bits = 0;
    c->cache_b = in->batch_stride;
    c->cache_h = in->head_stride;
    c->B = static_cast<int>(in->B);
    c->G = static_cast<int>(in->G);
    c->D = static_cast<int>(in->D);
    c->N = static_cast<int>(in->N);
    c->T = 0;
    c->at_once = 1;
    return in->B == 0 || in->N == 0 || in->G == 0 ||
           (in->k != nullptr && in->v != nullptr && in->k_scales != nullptr && in->v_scales != nullptr &&
            codes_aligned(in->k, in->k_scales, c->D) && codes_aligned(in->v, in->v_scales, c->D));
}

// Blocks of one key head's tokens; false if the launch would not hold them all.
bool blocks_of(const CacheCall& c, int tokens, uint32_t* each, uint32_t* all) {
    const int64_t n = (static_cast<int64_t>(tokens) + rows_of(c.D) - 1) / rows_of(c.D);
    const int64_t units = int64_t(2) * c.B * c.G;
    if (units > INT32_MAX || n > INT32_MAX / units) return false;
    *each = static_cast<uint32_t>(n);
    *all = static_cast<uint32_t>(n * units);
    return true;
}

template <typename F>
hipError_t with_type(int32_t type, int bits, F f) {
    auto of = [&](auto t) {
        return bits == 8 ? f(t, std::integral_constant<int, 8>{}) : f(t, std::integral_constant<int, 4>{});
    };
    switch (type) {
        case POINTOPS_F32: return of(float{});
        case POINTOPS_F16: return of(f16{});
        default: return of(bf16{});
    }
}

// Whether n values at p are whole words (of 16 bytes at most).
bool pieces(const void* p, int32_t type, int n) {
    return reinterpret_cast<uintptr_t>(p) % std::min(16, n * (type == POINTOPS_F32 ? 4 : 2)) == 0;
}

}  // namespace
}  // namespace attn
}  // namespace pointops

extern "C" {

hipError_t pointops_cache_write(const pointops_cache* cache, const void* k, const int64_t* k_stride, const void* v,
                                const int64_t* v_stride, int64_t tokens, const void* lengths, int32_t length_bits,
                                const void* starts, int32_t start_bits, int32_t type, hipStream_t stream) {
    using namespace pointops::attn;
    CacheCall c;
    if (!read_cache(cache, &c) || tokens < 0 || tokens > (int64_t(1) << 30) - 1024) return hipErrorInvalidValue;
    if (type < POINTOPS_F32 || type > POINTOPS_BF16) return hipErrorInvalidValue;
    if ((lengths != nullptr && length_bits != 32 && length_bits != 64) ||
        (starts != nullptr && start_bits != 32 && start_bits != 64))
        return hipErrorInvalidValue;
    if (c.B == 0 || c.G == 0 || c.N == 0 || tokens == 0) return hipSuccess;
    if (k == nullptr || v == nullptr || k_stride == nullptr || v_stride == nullptr) return hipErrorInvalidValue;
    for (int n : {4, 8}) {
        bool whole = pieces(k, type, n) && pieces(v, type, n) && c.D % n == 0;
        for (int i = 0; i < 3; ++i) whole = whole && k_stride[i] % n == 0 && v_stride[i] % n == 0;
        if (whole) c.at_once = n;
    }
    c.side[0].rows = k;
    c.side[1].rows = v;
    for (int i = 0; i < 2; ++i) {
        const int64_t* const stride = i == 0 ? k_stride : v_stride;
        c.side[i].b = stride[0];
        c.side[i].n = stride[1];
        c.side[i].h = stride[2];
    }
    c.lengths = lengths;
    c.starts = starts;
    c.length_bits = length_bits;
    c.start_bits = start_bits;
    c.T = static_cast<int>(tokens);
    uint32_t each, all;
    if (!blocks_of(c, c.T, &each, &all)) return hipErrorInvalidValue;
    return with_type(type, cache->bits, [&](auto t, auto bits) {
        return in_launches(all, [&](uint32_t first, uint32_t count) {
            hipLaunchKernelGGL((cache_write_kernel<decltype(t), decltype(bits)::value>), dim3(count), dim3(kThreads), 0, stream, c, each, first);
        });
    });
}

hipError_t pointops_cache_read(const pointops_cache* cache, void* k, void* v, int32_t type, hipStream_t stream) {
    using namespace pointops::attn;
    CacheCall c;
    if (!read_cache(cache, &c) || type < POINTOPS_F32 || type > POINTOPS_BF16) return hipErrorInvalidValue;
    if (c.B == 0 || c.G == 0 || c.N == 0) return hipSuccess;
    if (k == nullptr || v == nullptr) return hipErrorInvalidValue;
    for (int n : {4, 8})
        if (pieces(k, type, n) && pieces(v, type, n) && c.D % n == 0) c.at_once = n;
    uint32_t each, all;
    if (!blocks_of(c, c.N, &each, &all)) return hipErrorInvalidValue;
    return with_type(type, cache->bits, [&](auto t, auto bits) {
        using T = decltype(t);
        return in_launches(all, [&](uint32_t first, uint32_t count) {
            hipLaunchKernelGGL((cache_read_kernel<T, decltype(bits)::value>), dim3(count), dim3(kThreads), 0, stream, c,
                               static_cast<T*>(k), static_cast<T*>(v), each, first);
        });
    });
}

}  // extern "C"
