// The 4-bit form of cache rows.  Per 32 dims of a row one 16-bit word and 16
// bytes of codes c (0..15), two a byte, the low nibble the even dim's:
//   value = (c - z) * scale
// where the word is an fp16 scale of 7 significant bits, whose 4 low bits, which
// such a scale leaves free, hold the zero point z.  A value has at most 4 + 7 = 11
// significant bits, so it is an fp16 number as it stands: a cache of 4 bits feeds
// fp16 arithmetic with no further rounding.  0.5625 bytes a value.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device_common.hpp"

namespace asdsl {

constexpr int kGroup4 = 32;  // dims per scale word

typedef _Float16 half2_4 __attribute__((ext_vector_type(2)));

// Scale and zero point of two values' words (halves of `words`) as the pair
// arithmetic takes them.
struct Step4 {
    half2_4 scale, zero;  // zero: 1024 + z
    __device__ __forceinline__ explicit Step4(uint32_t words)
        : scale(__builtin_bit_cast(half2_4, words & 0xFFF0FFF0u)),
          zero(__builtin_bit_cast(half2_4, with_1024(words))) {}
    // The codes at bits 4 * i .. and 16 + 4 * i .. of w: 0x6400 | c is 1024 + c, the
    // difference is exact, and so is the product.
    __device__ __forceinline__ uint32_t values(uint32_t w, int i) const {
        return __builtin_bit_cast(uint32_t, (__builtin_bit_cast(half2_4, with_1024(w >> (4 * i))) - zero) * scale);
    }
    // The low 4 bits of both halves of w as fp16 numbers 1024 + c.  One instruction, which
    // takes one constant from a scalar register and the other from a vector one; left
    // to itself the compiler takes two with a literal each.
    static __device__ __forceinline__ uint32_t with_1024(uint32_t w) {
        uint32_t r;
        asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(w), "s"(0x000F000Fu), "v"(0x64006400u));
        return r;
    }
};

// A word of one row for both halves.
__device__ __forceinline__ uint32_t both4(uint32_t word) { return word | (word << 16); }

// One value from its code.
__device__ __forceinline__ float value4(uint32_t code, uint32_t word) {
    const _Float16 scale = __builtin_bit_cast(_Float16, static_cast<uint16_t>(word & 0xFFF0u));
    return static_cast<float>(static_cast<_Float16>(static_cast<int>(code) - static_cast<int>(word & 15u)) * scale);
}

// ----------------------------------------------------------------- quantizing
// In 64 bits throughout, so that a code or a scale next to a border of its
// rounding is the one that the definition in real numbers gives:
//   lo = min(0, x), hi = max(0, x) over the group, x held to +-2^15
//   scale = (hi - lo) / 15 rounded up to 7 significant bits, below 2^-14 to a
//           multiple of 2^-20, at least 2^-20
//   z = round-half-even(-lo / scale), c = clamp(round-half-even(x / scale) + z, 0, 15)
// A group with a value that is not finite has the scale NaN, so all of it reads as
// NaN.
constexpr double kMost4 = 32768.0;
constexpr uint32_t kNaN4 = 0x7E00u;

__device__ __forceinline__ double scale4(double range) {
    const double q = range / 15.0;
    if (q >= 0x1p-14) {
        const uint64_t low = (1ull << 46) - 1;  // of 52 mantissa bits 6 stay
        return __builtin_bit_cast(double, (__builtin_bit_cast(uint64_t, q) + low) & ~low);
    }
    return fmax(ceil(q * 0x1p20), 1.0) * 0x1p-20;
}

// The value of another lane of the same 8: lane ^ 1, lane ^ 2, the mirrored one.
template <int CTRL>
__device__ __forceinline__ double moved8(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), CTRL, 0xF, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, 0xF, 0xF, false);
    return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}

// Four neighbouring dims of a lane, a group's 32 in 8 neighbouring lanes, all of
// them here: the lane's codes (16 bits) and the group's word.  A quotient is formed
// in fp32, within 2^-18 of itself, and in fp64 only where that leaves its rounding
// open, some 4 in 10^5; with fp64 divisions throughout an append of 2045 tokens (8
// KV heads of 128) took 2 us more.
__device__ __forceinline__ uint32_t quantize4(const double (&x)[4], uint32_t& word) {
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const bool bad = !(isfinite(x[0]) && isfinite(x[1]) && isfinite(x[2]) && isfinite(x[3]));
    const uint64_t any = __builtin_amdgcn_ballot_w64(bad);
    double y[4], lo = 0.0, hi = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        y[i] = fmin(fmax(x[i], -kMost4), kMost4);
        lo = fmin(lo, y[i]);
        hi = fmax(hi, y[i]);
    }
    lo = fmin(lo, moved8<kDppQuadXor1>(lo));
    hi = fmax(hi, moved8<kDppQuadXor1>(hi));
    lo = fmin(lo, moved8<kDppQuadXor2>(lo));
    hi = fmax(hi, moved8<kDppQuadXor2>(hi));
    lo = fmin(lo, moved8<kDppRowHalfMirror>(lo));
    hi = fmax(hi, moved8<kDppRowHalfMirror>(hi));
    if (((any >> (lane & 56)) & 0xFFull) != 0ull) {
        word = kNaN4;
        return 0u;
    }
    const double scale = scale4(hi - lo);
    const float inv = 1.0f / static_cast<float>(scale);  // the scale is an fp32 number
    const auto rounded = [&](double v) {
        const float t = static_cast<float>(v) * inv;  // |t| < 17: off by less than 2^-18
        float r = __builtin_rintf(t);
        if (fabsf(fabsf(t - r) - 0.5f) < 0x1p-16f) r = static_cast<float>(rint(v / scale));
        return r;
    };
    const float zero = rounded(-lo);
    uint32_t codes = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        codes |= static_cast<uint32_t>(fminf(fmaxf(rounded(y[i]) + zero, 0.0f), 15.0f)) << (4 * i);
    const _Float16 h = static_cast<_Float16>(static_cast<float>(scale));  // exactly
    word = __builtin_bit_cast(uint16_t, h) | static_cast<uint32_t>(zero);
    return codes;
}

}  // namespace asdsl
