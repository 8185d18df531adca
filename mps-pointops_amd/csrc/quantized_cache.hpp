// Keys and values of a cache in 8 or 4 bits (gfx950).
//
// A row of D values is held as codes of P (D rounded up to a multiple of 32)
// values and a scale for each 32 of them:
//
//   X = 2^x, x the smallest whole number >= -127 with max |v| <= M X
//   code = v / X rounded to the nearest value of the type, even codes at ties
//
// 8 bits: E4M3 (1 sign, 4 exponent, 3 fraction bits; M = 448), 4 bits: E2M1
// (0, 0.5, 1, 1.5, 2, 3, 4, 6; M = 6); scales are bytes x + 127.  A group with an
// infinity or NaN has the scale 255 and reads as NaN.  Both are the block formats of
// the OCP Microscaling specification, which the card converts by instruction: two
// values at a time with their scale, exactly (compared for all codes and scales).
// A quotient by a power of two is exact, and so is all of this: the codes do not
// depend on how they are computed.  The last value of a 4-bit byte is its high half.
//
// Where the specification takes the exponent of the largest magnitude alone, so that
// magnitudes from 448 X (6 X) to 512 X (8 X) are cut to M, the scale here is twice as
// large for those groups and nothing is cut.
#pragma once

#include <algorithm>

#include "attention.hpp"

namespace pointops {
namespace attn {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

constexpr int kGroup = 32;      // values with a common scale
constexpr int kNoNumber = 255;  // the scale of a group with an infinity or NaN

__host__ __device__ constexpr int padded(int D) { return (D + kGroup - 1) / kGroup * kGroup; }

// A launch holds fewer than 2^32 threads: more than 2^23 blocks are several launches, each of
// `count` blocks from `first` on.
template <typename F>
hipError_t in_launches(uint32_t blocks, F launch) {
    constexpr uint32_t kMost = 1 << 23;
    for (uint32_t first = 0; first < blocks; first += kMost) {
        launch(first, std::min(kMost, blocks - first));
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

// Rows are read in pieces of up to 16 bytes, a row's 2 or 4 scales at once.
inline bool codes_aligned(const void* codes, const void* scales, int D) {
    const int each = padded(D) / kGroup;
    return reinterpret_cast<uintptr_t>(codes) % 16 == 0 && (each == 3 || reinterpret_cast<uintptr_t>(scales) % each == 0);
}

// A scale's byte as the conversions take it: they read the exponent field alone, in
// which 0 stands for 2^-127 and 255 for NaN.
__device__ __forceinline__ float scale_of(uint32_t byte) { return i2f(static_cast<int>(byte << 23)); }

// The byte of a group whose largest magnitude is `most`.
template <int BITS>
__device__ __forceinline__ uint32_t scale_byte(float most) {
    constexpr uint32_t kCarry = BITS == 8 ? 0x1fffff : 0x3fffff;  // a fraction above M's reaches the exponent
    constexpr int kTop = BITS == 8 ? 8 : 2;                       // M's exponent
    const uint32_t bits = static_cast<uint32_t>(f2i(most));
    if (bits >= 0x7f800000u) return kNoNumber;
    return static_cast<uint32_t>(max(static_cast<int>((bits + kCarry) >> 23) - kTop, 0));
}

// Two values of a word of codes: values 2 PAIR and 2 PAIR + 1, in bfloat16 and in 32 bits.
template <int BITS, int PAIR>
__device__ __forceinline__ int decode_bf16(uint32_t codes, float scale) {
    if constexpr (BITS == 8)
        return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, PAIR % 2 != 0));
    else
        return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, PAIR));
}
template <int BITS, int PAIR>
__device__ __forceinline__ f32x2 decode(uint32_t codes, float scale) {
    if constexpr (BITS == 8) return __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, scale, PAIR % 2 != 0);
    else return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, PAIR);
}

// Eight values' codes (8 bits: two words) as a fragment in bfloat16.
template <int BITS>
__device__ __forceinline__ i32x4 decode8(const uint32_t* codes, float scale) {
    if constexpr (BITS == 8)
        return i32x4{decode_bf16<8, 0>(codes[0], scale), decode_bf16<8, 1>(codes[0], scale),
                     decode_bf16<8, 0>(codes[1], scale), decode_bf16<8, 1>(codes[1], scale)};
    else
        return i32x4{decode_bf16<4, 0>(codes[0], scale), decode_bf16<4, 1>(codes[0], scale),
                     decode_bf16<4, 2>(codes[0], scale), decode_bf16<4, 3>(codes[0], scale)};
}

// Value `at` of a row.
template <int BITS>
__device__ __forceinline__ float decode_one(const uint8_t* row, const uint8_t* scales, int at) {
    const float scale = scale_of(scales[at / kGroup]);
    if constexpr (BITS == 8) return decode<8, 0>(row[at], scale)[0];
    else return decode<4, 0>(static_cast<uint32_t>(row[at / 2]) >> (at % 2 * 4), scale)[0];
}

}  // namespace attn
}  // namespace pointops
